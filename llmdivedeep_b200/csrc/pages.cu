// Pages of the paged caches: copying, giving to sequences, forking, freeing, compacting.
//
// State, all of it the caller's: refs[num_pages], how many sequences hold a page (0 = free); table[B, stride], the pages of a sequence in
// order, -1 behind the last one; ctx_len[B], its tokens.  A page holds 64 tokens.  Pages are taken lowest free id first, in the order
// of the call's list, so that ids depend on nothing but the state.  The calls that take pages are all or nothing: a bad argument (status
// 2) or too few free pages (status 3) leaves everything as it was.
//
// Who gets which page is decided by one cluster of CTAs that scan refs (each a stretch of it, counts exchanged through distributed
// shared memory); the contents are copied by a second kernel over the whole GPU, which starts under the first one's end.
#include "dsa_common.cuh"
#include "dsa_host.h"

namespace dsa {

constexpr int kPageTokens = 64;
constexpr int kPoolThreads = 1024, kPoolWarps = kPoolThreads / 32;
constexpr int kPoolCtas = 8;                           // the largest portable cluster
constexpr int kCopyThreads = 256, kCopyChunk = 16384;  // bytes of a page that a block copies at a time
constexpr int kCopyCaches = 128;                       // caches of one launch

// ---- one CTA, one cluster ------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
// every thread of the cluster; what was written before, to shared and to global memory, is seen after
__device__ __forceinline__ void pool_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int load_peer(const int* p, uint32_t cta) {
  uint32_t addr;
  int x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(cta));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
  return x;
}

struct PoolShared {
  int warp[kPoolWarps];
  int total;
  int count[4];                                        // what the CTAs of the cluster tell one another
};

// Exclusive prefix of v over the CTA's threads; the sum in `total`.  Every thread comes here.
__device__ __forceinline__ int block_prefix(PoolShared& s, int v, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                                     // the last call's results have been read
  if (lane == 31) s.warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const int w = s.warp[lane];
    int z = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += y;
    }
    s.warp[lane] = z - w;
    if (lane == 31) s.total = z;
  }
  __syncthreads();
  total = s.total;
  return s.warp[warp] + x - v;
}

// The stretch of the pool that this CTA scans: whole groups of four pages.
struct Stretch { int lo, hi; };
__device__ __forceinline__ Stretch my_stretch(int num_pages) {
  const int ctas = (int)cluster_size(), per = ((num_pages + ctas - 1) / ctas + 3) & ~3;
  const int64_t lo = (int64_t)cluster_rank() * per;
  return {(int)(lo < num_pages ? lo : num_pages), (int)(lo + per < num_pages ? lo + per : num_pages)};
}
// refs of pages p .. p + 3, p a multiple of four; pages past the pool count as held
__device__ __forceinline__ int4 refs4(const int32_t* refs, int p, int hi) {
  if (p + 4 <= hi && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) return *reinterpret_cast<const int4*>(refs + p);
  return make_int4(p < hi ? refs[p] : 1, p + 1 < hi ? refs[p + 1] : 1, p + 2 < hi ? refs[p + 2] : 1, p + 3 < hi ? refs[p + 3] : 1);
}

__device__ __forceinline__ int free_in(const int32_t* refs, Stretch st) {
  int n = 0;
  for (int p = st.lo + threadIdx.x * 4; p < st.hi; p += kPoolThreads * 4) {
    const int4 r = refs4(refs, p, st.hi);
    n += (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
  }
  return n;
}

// Free pages below this CTA's stretch and in the whole pool.  Every thread of the cluster comes here.
__device__ __forceinline__ void free_counts(PoolShared& s, const int32_t* refs, Stretch st, int& below, int& all) {
  int total;
  block_prefix(s, free_in(refs, st), total);
  if (threadIdx.x == 0) s.count[0] = total;
  pool_sync();
  below = all = 0;
  for (uint32_t c = 0; c < cluster_size(); ++c) {
    const int n = load_peer(&s.count[0], c);
    all += n;
    below += c < cluster_rank() ? n : 0;
  }
}

// The `want` lowest free pages: page of rank r -> fresh[r], and held once from here on.
__device__ __forceinline__ void take_pages(PoolShared& s, int32_t* refs, Stretch st, int below, int want, int32_t* fresh) {
  int base = below;
  for (int p0 = st.lo; p0 < st.hi && base < want; p0 += kPoolThreads * 4) {
    const int p = p0 + threadIdx.x * 4;
    const int4 r = p < st.hi ? refs4(refs, p, st.hi) : make_int4(1, 1, 1, 1);
    const int f[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
    int total, at = base + block_prefix(s, f[0] + f[1] + f[2] + f[3], total);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f[i]) {
        if (at < want) {
          fresh[at] = p + i;
          refs[p + i] = 1;
        }
        ++at;
      }
    base += total;
  }
}

__device__ __forceinline__ int pages_of(int tokens) { return (int)(((int64_t)tokens + kPageTokens - 1) / kPageTokens); }

// A row of the call's list, once: false where it is out of range or was named before.  `seen`: a bit for each row, in shared memory.
__device__ __forceinline__ bool name_row(uint32_t* seen, int row, int B) {
  if (row < 0 || row >= B) return false;
  const uint32_t bit = 1u << (row & 31);
  return (atomicOr(&seen[row >> 5], bit) & bit) == 0;
}

struct PoolArgs {
  int32_t* table;
  int64_t stride;
  int P, B;                                            // pages of a table row, rows
  int32_t* ctx;
  int32_t* refs;
  int num_pages, n;                                    // pages of the pool, entries of the list(s)
  const int32_t *a, *b;                                // extend: rows, n_new; fork: parents, children
  int max_new;                                         // extend
  int32_t* slots;                                      // extend: [n, max_new]
  int32_t *fresh, *first;                              // workspace: the pages taken, where entry i's begin
  int32_t *src, *dst, *tokens;                         // fork: what the copy kernel is to do
  int* status;
};

// ---- room for new tokens ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kPoolThreads) extend_kernel(const PoolArgs a) {
  __shared__ PoolShared s;
  extern __shared__ uint32_t seen[];
  const int gthread = cluster_rank() * kPoolThreads + threadIdx.x, gthreads = cluster_size() * kPoolThreads;
  for (int i = threadIdx.x; i < (a.B + 31) / 32; i += kPoolThreads) seen[i] = 0;
  __syncthreads();
  // every CTA looks the whole list over; where an entry's pages begin is written down by the first
  bool bad = false;
  int64_t want = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPoolThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < a.n) {
      const int row = a.a[i], nn = a.b[i];
      const int c = name_row(seen, row, a.B) ? a.ctx[row] : -1;
      if (c < 0 || nn < 0 || nn > a.max_new || (int64_t)c + nn > (int64_t)a.P * kPageTokens) bad = true;
      else need = pages_of(c + nn) - pages_of(c);
    }
    int total;
    const int at = block_prefix(s, need, total);
    if (i < a.n && cluster_rank() == 0 && want + at < a.num_pages) a.first[i] = (int)want + at;
    want += total;
  }
  bad = __syncthreads_or(bad);
  const Stretch st = my_stretch(a.num_pages);
  int below, all;
  free_counts(s, a.refs, st, below, all);
  const bool refused = bad || want > all;
  if (refused && gthread == 0 && a.status) atomicCAS(a.status, kStatusOk, bad ? kStatusBadIndex : kStatusNoPages);
  if (!refused) take_pages(s, a.refs, st, below, (int)want, a.fresh);
  pool_sync();
  // a warp per page that an entry's new tokens lie in
  const int lane = threadIdx.x & 31, per = (int)(((int64_t)a.max_new + 2 * kPageTokens - 2) / kPageTokens);
  for (int64_t u = gthread >> 5; u < (int64_t)a.n * per; u += gthreads >> 5) {
    const int i = (int)(u / per);
    int32_t* out = a.slots + (int64_t)i * a.max_new;
    if (refused) {                                     // nothing is written through them
      for (int t = (int)(u % per) * kPageTokens + lane; t < min(a.max_new, (int)(u % per + 1) * kPageTokens); t += 32) out[t] = -1;
      continue;
    }
    const int row = a.a[i], nn = a.b[i], c = a.ctx[row], held = pages_of(c), p = c / kPageTokens + (int)(u % per);
    int32_t* trow = a.table + (int64_t)row * a.stride;
    int page = -1;
    if (p < pages_of(c + nn)) {
      page = p < held ? trow[p] : a.fresh[a.first[i] + p - held];
      if (p >= held && lane == 0) trow[p] = page;
    }
    for (int k = lane; k < kPageTokens; k += 32) {     // places past the new tokens: -1
      const int64_t t = (int64_t)p * kPageTokens + k - c;
      if (t >= 0 && t < a.max_new) out[t] = t < nn && page >= 0 ? page * kPageTokens + k : -1;
    }
  }
  pool_sync();                                         // everyone has read ctx
  if (!refused)
    for (int i = gthread; i < a.n; i += gthreads) a.ctx[a.a[i]] += a.b[i];
}

// ---- forks -----------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kPoolThreads) fork_kernel(const PoolArgs a) {
  __shared__ PoolShared s;
  extern __shared__ uint32_t seen[];
  launch_dependents();
  const int gthread = cluster_rank() * kPoolThreads + threadIdx.x, gthreads = cluster_size() * kPoolThreads;
  for (int i = threadIdx.x; i < (a.B + 31) / 32; i += kPoolThreads) seen[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < a.n; i += kPoolThreads) {
    const int child = a.b[i];
    if (!name_row(seen, child, a.B) || a.ctx[child] != 0) bad = true;
  }
  __syncthreads();
  int64_t want = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPoolThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < a.n) {
      const int parent = a.a[i];
      if (parent < 0 || parent >= a.B || (seen[parent >> 5] >> (parent & 31) & 1u)) {
        bad = true;
      } else {
        const int c = a.ctx[parent];
        if (c < 0 || (int64_t)c > (int64_t)a.P * kPageTokens) bad = true;
        else need = c % kPageTokens != 0;
      }
    }
    int total;
    const int at = block_prefix(s, need, total);
    if (i < a.n && cluster_rank() == 0) a.first[i] = (int)want + at;
    want += total;
  }
  bad = __syncthreads_or(bad);
  const Stretch st = my_stretch(a.num_pages);
  int below, all;
  free_counts(s, a.refs, st, below, all);
  const bool refused = bad || want > all;
  if (refused) {
    if (gthread == 0 && a.status) atomicCAS(a.status, kStatusOk, bad ? kStatusBadIndex : kStatusNoPages);
    for (int i = gthread; i < a.n; i += gthreads) a.src[i] = -1;
    pool_sync();                                       // nobody leaves while its count may still be read
    return;
  }
  take_pages(s, a.refs, st, below, (int)want, a.fresh);
  pool_sync();
  // a warp per 32 pages of a fork
  const int lane = threadIdx.x & 31, per = (a.P + 31) / 32;
  for (int64_t u = gthread >> 5; u < (int64_t)a.n * per; u += gthreads >> 5) {
    const int i = (int)(u / per), p = (int)(u % per) * 32 + lane, c = a.ctx[a.a[i]], whole = c / kPageTokens;
    if (p >= a.P) continue;
    const int32_t* from = a.table + (int64_t)a.a[i] * a.stride;
    int32_t* to = a.table + (int64_t)a.b[i] * a.stride;
    int page = -1;
    if (p < whole) {
      page = from[p];
      if (page >= 0 && page < a.num_pages) atomicAdd(&a.refs[page], 1);
      else if (a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
    } else if (p == whole && c % kPageTokens) {
      page = a.fresh[a.first[i]];
    }
    to[p] = page;
  }
  pool_sync();                                         // everyone has read ctx
  for (int i = gthread; i < a.n; i += gthreads) {
    const int parent = a.a[i], c = a.ctx[parent], rest = c % kPageTokens;
    a.ctx[a.b[i]] = c;
    a.tokens[i] = rest;
    a.src[i] = rest ? a.table[(int64_t)parent * a.stride + c / kPageTokens] : -1;
    a.dst[i] = rest ? a.fresh[a.first[i]] : -1;
  }
}

// ---- freeing: a CTA per row ------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) free_kernel(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages,
                                                   const int32_t* rows, int* status) {
  __shared__ int tokens;
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= B) {
    if (threadIdx.x == 0 && status) atomicCAS(status, kStatusOk, kStatusBadIndex);
    return;
  }
  if (threadIdx.x == 0) tokens = atomicExch(&ctx[row], 0);         // a row that is named twice is empty the second time
  __syncthreads();
  const int n = min(pages_of(max(tokens, 0)), P);
  for (int p = threadIdx.x; p < n; p += blockDim.x) {
    int32_t* entry = table + (int64_t)row * stride + p;
    const int page = *entry;
    *entry = -1;
    if (page >= 0 && page < num_pages) {
      if (atomicSub(&refs[page], 1) > 0) continue;
      atomicAdd(&refs[page], 1);                       // was free already: the state is not what it says
    }
    if (status) atomicCAS(status, kStatusOk, kStatusBadIndex);
  }
}

// ---- compacting ------------------------------------------------------------------------------------------------------
struct CompactArgs {
  const int32_t* refs;
  int32_t* new_refs;
  int num_pages;
  int32_t *hi, *hi_refs, *lo, *remap;                  // workspace: pages to move (highest first), places for them (lowest first), new ids from L on
  int32_t* count;                                      // [2]: pages that move, L
};

// L pages are in use.  The i-th highest of them, from page L on, goes to the i-th lowest free page, below L: the pages that move and the
// places that take them have nothing in common, so all can be copied at once.
__global__ void __launch_bounds__(kPoolThreads) compact_kernel(const CompactArgs a) {
  __shared__ PoolShared s;
  launch_dependents();
  const int gthread = cluster_rank() * kPoolThreads + threadIdx.x, gthreads = cluster_size() * kPoolThreads;
  const Stretch st = my_stretch(a.num_pages);
  int below, all;
  free_counts(s, a.refs, st, below, all);
  const int L = a.num_pages - all;
  int free_base = below, holes = 0;
  for (int p0 = st.lo; p0 < st.hi; p0 += kPoolThreads * 4) {
    const int p = p0 + threadIdx.x * 4;
    const int4 r4 = p < st.hi ? refs4(a.refs, p, st.hi) : make_int4(1, 1, 1, 1);
    const int r[4] = {r4.x, r4.y, r4.z, r4.w};
    int total, at = free_base + block_prefix(s, (r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0), total);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = p + i;
      if (q >= st.hi) break;
      if (r[i] == 0) {
        if (q < L) {
          a.lo[at] = q;
          ++holes;
        } else {
          a.remap[q] = q;
          a.new_refs[q] = 0;
        }
        ++at;
      } else if (q < L) {
        a.new_refs[q] = r[i];
      } else {
        const int k = L - 1 - (q - at);                // q - at pages in use lie below this one
        a.hi[k] = q;
        a.hi_refs[k] = r[i];
        a.new_refs[q] = 0;
      }
    }
    free_base += total;
  }
  int mine;
  block_prefix(s, holes, mine);
  if (threadIdx.x == 0) s.count[1] = mine;
  pool_sync();
  int moves = 0;
  for (uint32_t c = 0; c < cluster_size(); ++c) moves += load_peer(&s.count[1], c);
  for (int k = gthread; k < moves; k += gthreads) {
    a.remap[a.hi[k]] = a.lo[k];
    a.new_refs[a.lo[k]] = a.hi_refs[k];
  }
  if (gthread == 0) {
    a.count[0] = moves;
    a.count[1] = L;
  }
  pool_sync();                                         // nobody leaves while a count may still be read
}

// ---- contents --------------------------------------------------------------------------------------------------------
struct CacheEntry {
  uint8_t* base;
  int64_t layer_stride;                                // bytes
  int32_t layers, token_bytes;
};
struct CopyArgs {
  CacheEntry cache[kCopyCaches];
  int32_t first[kCopyCaches + 1];                      // chunks of one page in the caches before
  int n_caches, num_pages;
  const int32_t *src, *dst, *tokens;                   // tokens: null = whole pages
  const int32_t* count;                                // on the device; null: n
  int n;
  // compacting: the table is rewritten on the way
  const int32_t *table, *remap;
  int32_t* new_table;
  int64_t stride, new_stride;
  int B, P;
  int* status;
};

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyArgs a) {
  const int32_t *src = grid_wait(a.src), *dst = a.dst, *tokens = a.tokens;
  const int n = a.count ? *grid_wait(a.count) : a.n;
  if (a.table) {
    const int32_t* remap = grid_wait(a.remap);
    const int L = grid_wait(a.count)[1];
    for (int64_t e = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; e < (int64_t)a.B * a.P; e += (int64_t)gridDim.x * kCopyThreads) {
      const int64_t b = e / a.P, p = e % a.P;
      const int page = a.table[b * a.stride + p];
      a.new_table[b * a.new_stride + p] = page >= L && page < a.num_pages ? remap[page] : page;
    }
  }
  const int chunks = a.first[a.n_caches];
  for (int64_t item = blockIdx.x; item < (int64_t)n * chunks; item += gridDim.x) {
    const int i = (int)(item / chunks), c = (int)(item % chunks);
    const int from = src[i], to = dst[i];
    if (from < 0 || to < 0) continue;                  // an entry that is not to be copied
    if (from >= a.num_pages || to >= a.num_pages) {
      if (threadIdx.x == 0 && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
      continue;
    }
    int e = 0;
    for (int hi = a.n_caches; hi - e > 1;) {           // the cache that chunk c belongs to
      const int mid = (e + hi) / 2;
      (c >= a.first[mid] ? e : hi) = mid;
    }
    const CacheEntry& ce = a.cache[e];
    const int page_bytes = kPageTokens * ce.token_bytes, per = (page_bytes + kCopyChunk - 1) / kCopyChunk;
    const int in = c - a.first[e], layer = in / per, b0 = in % per * kCopyChunk;
    const int bytes = tokens ? min(max(tokens[i], 0), kPageTokens) * ce.token_bytes : page_bytes;
    const int len = min(bytes - b0, kCopyChunk);
    if (len <= 0) continue;
    const uint8_t* f = ce.base + layer * ce.layer_stride + (int64_t)from * page_bytes + b0;
    uint8_t* d = ce.base + layer * ce.layer_stride + (int64_t)to * page_bytes + b0;
    for (int o = threadIdx.x * 16; o + 16 <= len; o += kCopyThreads * 16) *reinterpret_cast<uint4*>(d + o) = *reinterpret_cast<const uint4*>(f + o);
    const int rest = len & ~15, w = rest + threadIdx.x * 4;      // a token's bytes are a multiple of four
    if (w < len) *reinterpret_cast<uint32_t*>(d + w) = *reinterpret_cast<const uint32_t*>(f + w);
  }
}

// ---- launches --------------------------------------------------------------------------------------------------------
template <typename... Params, typename... Args>
static void launch_pool(void (*kern)(Params...), int num_pages, size_t smem, cudaStream_t stream, Args... args) {
  const int ctas = min(kPoolCtas, max(1, num_pages / (4 * kPoolThreads)));      // at least one turn of the scan for each
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPoolThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...);      // its error is the launch check's
}

static size_t seen_bytes(int B) { return (size_t)(B + 31) / 32 * 4; }

// Caches in groups that fit one launch; a.src and what else says which pages is set.  `most`: no more pages than that are copied.
static int launch_copies(CopyArgs& a, const dsa_page_cache* caches, int n_caches, int64_t most, int behind_plan, cudaStream_t stream) {
  int c0 = 0;
  do {
    a.n_caches = min(n_caches - c0, kCopyCaches);
    a.first[0] = 0;
    for (int c = 0; c < a.n_caches; ++c) {
      const dsa_page_cache& h = caches[c0 + c];
      a.cache[c] = {static_cast<uint8_t*>(h.base), h.layer_stride, h.layers, h.token_bytes};
      a.first[c + 1] = a.first[c] + h.layers * ((kPageTokens * h.token_bytes + kCopyChunk - 1) / kCopyChunk);
    }
    const int64_t items = max(most * a.first[a.n_caches], a.table ? ((int64_t)a.B * a.P + kCopyThreads - 1) / kCopyThreads : 0);
    const int grid = (int)min(items, (int64_t)sm_count() * 8);
    if (grid > 0) launch_after(behind_plan && c0 == 0, copy_kernel, dim3(grid), kCopyThreads, 0, stream, a);
    a.table = nullptr;                                 // rewritten once
    c0 += kCopyCaches;
  } while (c0 < n_caches);
  return check_launch("copy_pages");
}

int copy_pages_launch(const dsa_page_cache* caches, int n_caches, int num_pages, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n,
                      int32_t* status, cudaStream_t stream) {
  CopyArgs a{};
  a.num_pages = num_pages;
  a.src = src; a.dst = dst; a.tokens = tokens;
  a.n = n;
  a.status = status;
  return launch_copies(a, caches, n_caches, n, 0, stream);
}

static PoolArgs pool_args(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, int n, int32_t* status) {
  PoolArgs a{};
  a.table = table; a.stride = stride; a.P = P; a.B = B;
  a.ctx = ctx; a.refs = refs; a.num_pages = num_pages; a.n = n;
  a.status = status;
  return a;
}

// What the calls that take or move pages need: extend the pages taken and a place for each entry, fork those and what to copy,
// compact four lists of pages.
size_t pages_workspace_bytes(int num_pages, int n) { return ((size_t)4 * num_pages + (size_t)5 * n + 4) * sizeof(int32_t); }

int extend_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* rows, const int32_t* n_new, int n,
                        int max_new, int32_t* slots, int32_t* workspace, int32_t* status, cudaStream_t stream) {
  PoolArgs a = pool_args(table, stride, P, B, ctx, refs, num_pages, n, status);
  a.a = rows; a.b = n_new;
  a.max_new = max_new;
  a.slots = slots;
  a.first = workspace;
  a.fresh = workspace + n;
  launch_pool(extend_kernel, num_pages, seen_bytes(B), stream, a);
  return check_launch("extend_pages");
}

int fork_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* parents, const int32_t* children,
                      int n, const dsa_page_cache* caches, int n_caches, int32_t* workspace, int32_t* status, cudaStream_t stream) {
  PoolArgs a = pool_args(table, stride, P, B, ctx, refs, num_pages, n, status);
  a.a = parents; a.b = children;
  a.first = workspace;
  a.fresh = a.first + n;
  a.src = a.fresh + n;
  a.dst = a.src + n;
  a.tokens = a.dst + n;
  launch_pool(fork_kernel, num_pages, seen_bytes(B), stream, a);
  if (n_caches == 0) return check_launch("fork_pages");
  CopyArgs c{};
  c.num_pages = num_pages;
  c.src = a.src; c.dst = a.dst; c.tokens = a.tokens;
  c.n = n;
  c.status = status;
  return launch_copies(c, caches, n_caches, n, 1, stream);
}

int free_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* rows, int n, int32_t* status,
                      cudaStream_t stream) {
  free_kernel<<<n, 256, 0, stream>>>(table, stride, P, B, ctx, refs, num_pages, rows, status);
  return check_launch("free_pages");
}

int compact_pages_launch(const int32_t* table, int64_t stride, int32_t* new_table, int64_t new_stride, int P, int B, const int32_t* refs, int32_t* new_refs,
                         int num_pages, const dsa_page_cache* caches, int n_caches, int32_t* workspace, int32_t* status, cudaStream_t stream) {
  CompactArgs a{};
  a.refs = refs; a.new_refs = new_refs; a.num_pages = num_pages;
  a.count = workspace;
  a.hi = workspace + 4;
  a.hi_refs = a.hi + num_pages;
  a.lo = a.hi_refs + num_pages;
  a.remap = a.lo + num_pages;
  launch_pool(compact_kernel, num_pages, 0, stream, a);
  CopyArgs c{};
  c.num_pages = num_pages;
  c.src = a.hi; c.dst = a.lo;
  c.count = a.count;
  c.table = table; c.new_table = new_table; c.remap = a.remap;
  c.stride = stride; c.new_stride = new_stride; c.B = B; c.P = P;
  c.status = status;
  return launch_copies(c, caches, n_caches, num_pages / 2, 1, stream);
}

}  // namespace dsa
