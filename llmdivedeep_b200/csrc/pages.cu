// Pages of the paged caches: copying, giving to sequences, forking, freeing, compacting.
//
// State, all of it the caller's: refs[num_pages], how many sequences hold a page (0 = free); table[B, stride], the pages of a sequence in
// order, -1 behind the last one; ctx_len[B], its tokens.  A page holds 64 tokens.  Pages are taken lowest free id first, in the order
// of the call's list, so that ids depend on nothing but the state.  The calls that take pages are all or nothing: a bad argument, a partly filled
// last page that they copy or fill and that is no page (status 2), or too few free pages (status 3) leaves everything as it was.  Of full
// pages the table is believed: a fork copies an entry that is no page as it stands, and says so (status 2).
//
// Who gets which page is decided by one cluster of CTAs that scan refs (each a stretch of it, counts exchanged through distributed
// shared memory).  What is long goes to a second kernel over the whole GPU, which starts under the first one's end: the contents, the rows
// of forks, many slots.  These calls wait: for a launch, for loads that depend on one another, for barriers; only the contents have
// a bandwidth.
#include "dsa_common.cuh"
#include "dsa_host.h"

namespace dsa {

constexpr int kPageTokens = 64;
constexpr int kPoolThreads = 1024, kPoolWarps = kPoolThreads / 32;
constexpr int kPoolCtas = 8;                           // the largest portable cluster
constexpr int kCopyThreads = 128, kCopyCtas = 2;       // CTAs of an SM
constexpr int kCopyChunk = 16384, kCopyStages = 6, kCopyAhead = 3;      // bytes of a copy at most; stages; loads under way
constexpr int kCopySmem = kCopyStages * kCopyChunk + 128;
constexpr int kCopyCaches = 128;                       // caches of one launch
constexpr int kFillUnits = 512;                        // pages of new tokens up to which the planning cluster writes their slots itself

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
  if (cluster_size() == 1) {                           // most pools: a barrier of the cluster takes a microsecond more
    __syncthreads();
    return;
  }
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
  int warp[2][kPoolWarps];
  int count[2];                                        // what the CTAs of the cluster tell one another
};

__device__ __forceinline__ int warp_inclusive(int x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}
// Exclusive prefix of v over the CTA's threads; the sum in `total`.  Every thread comes here, `turn` counts the calls: they take the two
// rows of s.warp in turn, so that one barrier a call is enough.
__device__ __forceinline__ int block_prefix(PoolShared& s, int& turn, int v, int& total) {
  int* row = s.warp[turn++ & 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, x = warp_inclusive(v);
  if (lane == 31) row[warp] = x;
  __syncthreads();
  const int w = row[lane], z = warp_inclusive(w);
  total = __shfl_sync(0xffffffffu, z, 31);
  return __shfl_sync(0xffffffffu, z - w, warp) + x - v;
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

// The four pages of this thread in the first turn over the stretch, requested before anything else is done.
__device__ __forceinline__ int4 first_refs(const int32_t* refs, Stretch st) {
  const int p = st.lo + threadIdx.x * 4;
  return p < st.hi ? refs4(refs, p, st.hi) : make_int4(1, 1, 1, 1);
}
__device__ __forceinline__ int free_of(int4 r) { return (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0); }
__device__ __forceinline__ int free_in(const int32_t* refs, Stretch st, int4 first) {
  int n = free_of(first);
  for (int p = st.lo + (kPoolThreads + threadIdx.x) * 4; p < st.hi; p += kPoolThreads * 4) n += free_of(refs4(refs, p, st.hi));
  return n;
}

// s.count[which] of the CTAs below this one, and of all.  Every thread of the cluster comes here after a pool_sync.
__device__ __forceinline__ void sum_counts(PoolShared& s, int which, int& below, int& all) {
  const int lane = threadIdx.x & 31, n = lane < (int)cluster_size() ? load_peer(&s.count[which], lane) : 0;      // eight at most
  all = __reduce_add_sync(0xffffffffu, n);
  below = __reduce_add_sync(0xffffffffu, lane < (int)cluster_rank() ? n : 0);
}
// Free pages below this CTA's stretch and in the whole pool.  Every thread of the cluster comes here.
__device__ __forceinline__ void free_counts(PoolShared& s, int& turn, const int32_t* refs, Stretch st, int4 first, int& below, int& all) {
  int total;
  block_prefix(s, turn, free_in(refs, st, first), total);
  if (threadIdx.x == 0) s.count[0] = total;
  pool_sync();
  sum_counts(s, 0, below, all);
}

// The `want` lowest free pages: page of rank r -> fresh[r], and held once from here on.
__device__ __forceinline__ void take_pages(PoolShared& s, int& turn, int32_t* refs, Stretch st, int4 first, int below, int want, int32_t* fresh) {
  int base = below;
  for (int p0 = st.lo; p0 < st.hi && base < want; p0 += kPoolThreads * 4) {
    const int p = p0 + threadIdx.x * 4;
    const int4 r = p0 == st.lo ? first : p < st.hi ? refs4(refs, p, st.hi) : make_int4(1, 1, 1, 1);
    const int f[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
    int total, at = base + block_prefix(s, turn, free_of(r), total);
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
  int32_t *refused, *fresh, *first;                    // workspace: whether nothing is done, the pages taken, where entry i's begin
  int32_t* held;                                       // extend: tokens of the rows before
  int32_t *src, *dst, *tokens;                         // fork: what the copy kernel is to do
  int fill;                                            // extend: the planning cluster writes the slots
  int* status;
};

// Whether entry p of a row names a page of the pool.
__device__ __forceinline__ bool names_page(const PoolArgs& a, int row, int p) { return (unsigned)a.table[(int64_t)row * a.stride + p] < (unsigned)a.num_pages; }

// ---- room for new tokens ---------------------------------------------------------------------------------------------
// Pages that an entry's new tokens lie in, at most
__host__ __device__ __forceinline__ int64_t extend_per(int max_new) { return ((int64_t)max_new + 2 * kPageTokens - 2) / kPageTokens; }
// Table entries and slots of the u-th such page of all: a warp's work.
__device__ __forceinline__ void extend_fill(const PoolArgs& a, int64_t u, int per, bool refused) {
  const int lane = threadIdx.x & 31, i = (int)(u / per), k0 = (int)(u - (int64_t)i * per);
  int32_t* out = a.slots + (int64_t)i * a.max_new;
  if (refused) {                                       // nothing is to be written through them
    for (int t = k0 * kPageTokens + lane; t < min(a.max_new, (k0 + 1) * kPageTokens); t += 32) out[t] = -1;
    return;
  }
  const int row = a.a[i], nn = a.b[i], c = a.held[i], first = a.first[i], held = pages_of(c), p = c / kPageTokens + k0;
  int32_t* trow = a.table + (int64_t)row * a.stride;
  int page = -1;
  if (p < pages_of(c + nn)) {
    page = p < held ? trow[p] : a.fresh[first + p - held];
    if (p >= held && lane == 0) trow[p] = page;
  }
#pragma unroll
  for (int k = lane; k < kPageTokens; k += 32) {       // places past the new tokens: -1
    const int64_t t = (int64_t)p * kPageTokens + k - c;
    if (t >= 0 && t < a.max_new) out[t] = t < nn && page >= 0 ? page * kPageTokens + k : -1;
  }
}

// 6.5 us with up to 2047 pages in the pool (9.3 with refs read after the list and cluster barriers throughout): loads that depend on one another.
__global__ void __launch_bounds__(kPoolThreads) extend_kernel(const PoolArgs a) {
  __shared__ PoolShared s;
  extern __shared__ uint32_t seen[];
  launch_dependents();
  int turn = 0;
  const int gthread = cluster_rank() * kPoolThreads + threadIdx.x, gthreads = cluster_size() * kPoolThreads;
  const Stretch st = my_stretch(a.num_pages);
  const int4 refs0 = first_refs(a.refs, st);
  for (int i = threadIdx.x; i < (a.B + 31) / 32; i += kPoolThreads) seen[i] = 0;
  __syncthreads();
  // every CTA looks the whole list over; what is learnt of an entry is written down by the first
  bool bad = false;
  int64_t want = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPoolThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0, c = -1;
    if (i < a.n) {
      const int row = a.a[i], nn = a.b[i];
      if (name_row(seen, row, a.B)) c = a.ctx[row];
      if (c < 0 || nn < 0 || nn > a.max_new || (int64_t)c + nn > (int64_t)a.P * kPageTokens) {
        bad = true;
      } else {
        need = pages_of(c + nn) - pages_of(c);
        if (nn > 0 && c % kPageTokens && !names_page(a, row, c / kPageTokens)) bad = true;      // the first new token goes there
      }
    }
    int total;
    const int at = block_prefix(s, turn, need, total);
    if (i < a.n && cluster_rank() == 0) {
      a.first[i] = (int)min(want + at, (int64_t)a.num_pages);
      a.held[i] = c;
    }
    want += total;
  }
  bad = __syncthreads_or(bad);
  int below, all;
  free_counts(s, turn, a.refs, st, refs0, below, all);
  const bool refused = bad || want > all;
  if (gthread == 0) {
    *a.refused = refused;
    if (refused && a.status) atomicCAS(a.status, kStatusOk, bad ? kStatusBadIndex : kStatusNoPages);
  }
  if (!refused) {
    for (int i = gthread; i < a.n; i += gthreads) a.ctx[a.a[i]] = a.held[i] + a.b[i];      // every CTA has read it: that was before the last barrier
    take_pages(s, turn, a.refs, st, refs0, below, (int)want, a.fresh);
  }
  pool_sync();                                         // the pages are known; and nobody leaves while its count may still be read
  if (!a.fill) return;
  const int per = (int)extend_per(a.max_new);
  for (int64_t u = gthread >> 5; u < (int64_t)a.n * per; u += gthreads >> 5) extend_fill(a, u, per, refused);
}
// 40 rows of up to 8320 new tokens: 35 us with the slots written by the cluster of six CTAs.
__global__ void __launch_bounds__(256) extend_fill_kernel(const PoolArgs a) {
  const bool refused = *grid_wait(a.refused) != 0;
  const int per = (int)extend_per(a.max_new);
  for (int64_t u = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5; u < (int64_t)a.n * per; u += gridDim.x * 8) extend_fill(a, u, per, refused);
}

// ---- forks -----------------------------------------------------------------------------------------------------------
// Who gets the pages, and what is to be copied; the rows of the children are the copy kernel's work.  5.2 us (7.7 before the same changes).
__global__ void __launch_bounds__(kPoolThreads) fork_kernel(const PoolArgs a) {
  __shared__ PoolShared s;
  extern __shared__ uint32_t seen[];
  launch_dependents();
  int turn = 0;
  const int gthread = cluster_rank() * kPoolThreads + threadIdx.x, gthreads = cluster_size() * kPoolThreads;
  const Stretch st = my_stretch(a.num_pages);
  const int4 refs0 = first_refs(a.refs, st);
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
        if (c < 0 || (int64_t)c > (int64_t)a.P * kPageTokens || (c % kPageTokens && !names_page(a, parent, c / kPageTokens))) bad = true;
        else need = c % kPageTokens;
      }
    }
    int total;
    const int at = block_prefix(s, turn, need != 0, total);
    if (i < a.n && cluster_rank() == 0) {
      a.first[i] = (int)want + at;
      a.tokens[i] = need;
    }
    want += total;
  }
  bad = __syncthreads_or(bad);
  int below, all;
  free_counts(s, turn, a.refs, st, refs0, below, all);
  const bool refused = bad || want > all;
  if (gthread == 0) {
    *a.refused = refused;
    if (refused && a.status) atomicCAS(a.status, kStatusOk, bad ? kStatusBadIndex : kStatusNoPages);
  }
  if (!refused) take_pages(s, turn, a.refs, st, refs0, below, (int)want, a.fresh);
  pool_sync();                                         // the pages are known; and nobody leaves while its count may still be read
  for (int i = gthread; i < a.n; i += gthreads) {
    const bool copied = !refused && a.tokens[i] != 0;
    a.src[i] = copied ? a.table[(int64_t)a.a[i] * a.stride + a.ctx[a.a[i]] / kPageTokens] : -1;
    a.dst[i] = copied ? a.fresh[a.first[i]] : -1;
  }
}
// 32 entries of a child's row: a warp's work.  Parents are no children, so their rows and lengths stay as they are meanwhile.
__device__ __forceinline__ void fork_row(const PoolArgs& a, int64_t u, int per) {
  const int lane = threadIdx.x & 31, i = (int)(u / per), p = (int)(u - (int64_t)i * per) * 32 + lane;
  const int parent = a.a[i], child = a.b[i], c = a.ctx[parent], whole = c / kPageTokens;
  if (u == (int64_t)i * per && lane == 0) a.ctx[child] = c;
  if (p >= a.P) return;
  int page = -1;
  if (p < whole) {
    page = a.table[(int64_t)parent * a.stride + p];
    if (page >= 0 && page < a.num_pages) atomicAdd(&a.refs[page], 1);
    else if (a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
  } else if (p == whole && c % kPageTokens) {
    page = a.dst[i];
  }
  a.table[(int64_t)child * a.stride + p] = page;
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
// places that take them have nothing in common, so all can be copied at once.  6000 pages: 7.7 us, of which the counting of what is used, then
// of what moves, are two passes.
__global__ void __launch_bounds__(kPoolThreads) compact_kernel(const CompactArgs a) {
  __shared__ PoolShared s;
  launch_dependents();
  int turn = 0;
  const int gthread = cluster_rank() * kPoolThreads + threadIdx.x, gthreads = cluster_size() * kPoolThreads;
  const Stretch st = my_stretch(a.num_pages);
  const int4 refs0 = first_refs(a.refs, st);
  int below, all;
  free_counts(s, turn, a.refs, st, refs0, below, all);
  const int L = a.num_pages - all;
  int free_base = below, holes = 0;
  for (int p0 = st.lo; p0 < st.hi; p0 += kPoolThreads * 4) {
    const int p = p0 + threadIdx.x * 4;
    const int4 r4 = p0 == st.lo ? refs0 : p < st.hi ? refs4(a.refs, p, st.hi) : make_int4(1, 1, 1, 1);
    const int r[4] = {r4.x, r4.y, r4.z, r4.w};
    int total, at = free_base + block_prefix(s, turn, free_of(r4), total);
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
  int mine, moves;
  block_prefix(s, turn, holes, mine);
  if (threadIdx.x == 0) s.count[1] = mine;
  pool_sync();
  sum_counts(s, 1, below, moves);
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
  int* status;
};
// What else the copy kernel does, by the warps that copy nothing.
enum CopyWork : int { kCopyOnly, kCopyFork, kCopyCompact };
struct RemapArgs {
  const int32_t *table, *remap, *count;
  int32_t* new_table;
  int64_t stride, new_stride;
  int B, P, num_pages;
};

// A page's chunk of one cache: global -> shared -> global memory by bulk copies, `kCopyAhead` loads under way while the ones before are
// stored, issued by one thread; each lane of its warp works out where one of the next 32 chunks is.  700 pages of 16 layers (785 MB moved): 126 us
// = 6.2 TB/s, the rate of a plain copy; 143 with a thread's loads and stores of 16 bytes, src and dst looked up chunk by chunk.
template <int WORK>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyArgs a, const PoolArgs f, const RemapArgs m) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kCopyStages * kCopyChunk);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(full + kCopyStages);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kCopyStages; ++i) mbar_init(full + i, 1);
    mbar_fence_init();
    *abort_flag = 0;
  }
  __syncthreads();
  if (warp > 0) {                                      // (grid_wait: what the planning kernel wrote)
    constexpr int kOthers = kCopyThreads - 32;
    if constexpr (WORK == kCopyFork) {
      if (*grid_wait(f.refused)) return;
      const int per = max(1, (f.P + 31) / 32);
      for (int64_t u = (int64_t)blockIdx.x * (kOthers / 32) + warp - 1; u < (int64_t)f.n * per; u += gridDim.x * (kOthers / 32)) fork_row(f, u, per);
    } else if constexpr (WORK == kCopyCompact) {
      const int L = grid_wait(m.count)[1];
      for (int64_t e = (int64_t)blockIdx.x * kOthers + threadIdx.x - 32; e < (int64_t)m.B * m.P; e += gridDim.x * kOthers) {
        const int64_t b = e / m.P, p = e - b * m.P;
        const int page = m.table[b * m.stride + p];
        m.new_table[b * m.new_stride + p] = page >= L && page < m.num_pages ? m.remap[page] : page;
      }
    }
    return;
  }
  const int32_t *src = grid_wait(a.src), *dst = a.dst, *tokens = a.tokens;
  const int n = a.count ? *grid_wait(a.count) : a.n, chunks = a.first[a.n_caches];
  const int64_t items = (int64_t)n * chunks;
  uint32_t loads = 0, stores = 0;                      // of this CTA, lane 0's
  uint64_t to[kCopyAhead] = {};                        // where the loads under way go, and how long they are
  uint32_t len[kCopyAhead] = {};
  bool ok = true;
  auto store_oldest = [&]() {                          // lane 0
    const uint32_t st = stores % kCopyStages;
    if (ok && !mbar_wait(full + st, (stores / kCopyStages) & 1, abort_flag, a.status)) ok = false;
    if (ok)
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;"
                   ::"l"(to[0]), "r"(smem_u32(smem + st * kCopyChunk)), "r"(len[0]) : "memory");
    ++stores;
#pragma unroll
    for (int i = 0; i + 1 < kCopyAhead; ++i) {
      to[i] = to[i + 1];
      len[i] = len[i + 1];
    }
  };
  for (int64_t item0 = blockIdx.x; item0 < items; item0 += (int64_t)gridDim.x * 32) {
    const int64_t item = item0 + (int64_t)lane * gridDim.x;
    uint64_t from_at = 0, to_at = 0;
    int bytes = 0;
    if (item < items) {
      const int i = (int)(item / chunks), c = (int)(item - (int64_t)i * chunks), from = src[i], to_page = dst[i];
      int e = 0;
      for (int hi = a.n_caches; hi - e > 1;) {         // the cache that chunk c belongs to
        const int mid = (e + hi) / 2;
        (c >= a.first[mid] ? e : hi) = mid;
      }
      const CacheEntry& ce = a.cache[e];
      const int page_bytes = kPageTokens * ce.token_bytes, per = (page_bytes + kCopyChunk - 1) / kCopyChunk;
      const int chunk = ((page_bytes + per - 1) / per + 15) & ~15, in = c - a.first[e], layer = in / per, b0 = (in - layer * per) * chunk;
      const int used = tokens ? min(max(tokens[i], 0), kPageTokens) * ce.token_bytes : page_bytes;
      if (from >= a.num_pages || to_page >= a.num_pages) {
        if (from >= 0 && to_page >= 0 && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
      } else if (from >= 0 && to_page >= 0) {          // a negative id: not to be copied
        bytes = max(0, min(used - b0, chunk));
        uint8_t* base = ce.base + layer * ce.layer_stride + b0;
        const uint8_t* s = base + (int64_t)from * page_bytes;
        uint8_t* d = base + (int64_t)to_page * page_bytes;
        for (int o = bytes & ~15; o < bytes; o += 4) *reinterpret_cast<uint32_t*>(d + o) = *reinterpret_cast<const uint32_t*>(s + o);      // a token's bytes are a multiple of four
        bytes &= ~15;
        from_at = reinterpret_cast<uint64_t>(s);
        to_at = reinterpret_cast<uint64_t>(d);
      }
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, bytes > 0); left; left &= left - 1) {
      const int who = __ffs(left) - 1;
      const uint64_t f_at = __shfl_sync(0xffffffffu, from_at, who), t_at = __shfl_sync(0xffffffffu, to_at, who);
      const uint32_t b = __shfl_sync(0xffffffffu, bytes, who);
      if (lane == 0) {
        if (loads - stores == kCopyAhead) store_oldest();
        // the stage's last store has been read: all but the latest kCopyStages - 1 - kCopyAhead
        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kCopyStages - 1 - kCopyAhead) : "memory");
        const uint32_t st = loads % kCopyStages;
        if (ok) {
          mbar_expect_tx(full + st, b);
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(smem_u32(smem + st * kCopyChunk)), "l"(f_at), "r"(b), "r"(smem_u32(full + st)) : "memory");
        }
#pragma unroll
        for (int i = 0; i < kCopyAhead; ++i)
          if (loads - stores == (uint32_t)i) {
            to[i] = t_at;
            len[i] = b;
          }
        ++loads;
      }
      __syncwarp();
    }
  }
  if (lane == 0) {
    while (stores < loads) store_oldest();
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // shared memory may go
    if (!ok)                                           // a wait gave up: let the copies in flight land (bounded)
      for (int w = 0; w < 64; ++w) __nanosleep(1000);
  }
}

// ---- acceptance of drafts ----------------------------------------------------------------------------------------------
// Row rows[i] keeps the drafts path[i, 0 .. n_keep[i]) of its last n_new[i] tokens: draft path[k] moves to place k behind the P tokens before
// them, in every cache; what lies behind goes.  path[k] >= k, so a place that is written is read by no later move, and a thread that takes
// the same 16 bytes of every token in order needs no barrier.  One CTA a row and 128 columns of 16 bytes; what bounds it is latency: list, table, then eight
// records under way at a time, and the pages in a second kernel, which starts under the first (200 rows x 16 layers 14.4 us).  Calls of up to eight rows whose columns
// are a CTA's threads are one cluster, and one launch: 8 rows x 2 layers 15.4 -> 13.8 us on the host, which the GPU's 8 wait for.
constexpr int kAcceptAlone = 8, kAcceptThreads = 1024;
template <int N>
struct AcceptCaches {                                  // of a launch; eight hold most models' in a tenth of the parameters
  CacheEntry cache[N];
  int32_t first[N + 1];                                // columns of one token in the caches before
  int n_caches;
};
struct AcceptArgs {
  int32_t *table, *ctx, *refs;
  int64_t stride;
  int P, B, num_pages, n;
  const int32_t *rows, *n_new, *path, *n_keep;
  int path_stride;
  int32_t* accepted;                                   // workspace [n]: whether row i is
  int* status;
};
// Whether entry i can be done; every thread of the CTA comes here.  A row is refused that the list has named before, whose numbers make no
// sense, whose drafts lie in pages that are none, or -- where something moves or goes -- whose kept drafts do in pages that others hold too.
__device__ __forceinline__ bool accept_valid(const AcceptArgs& a, int i) {
  const int row = a.rows[i], nn = a.n_new[i], keep = a.n_keep[i];
  bool bad = row < 0 || row >= a.B || nn < 0 || keep < 0 || keep > nn || keep > a.path_stride;
  const int c = bad ? 0 : a.ctx[row];
  if (c < nn || (int64_t)c > (int64_t)a.P * kPageTokens) bad = true;
  for (int j = threadIdx.x; j < i; j += blockDim.x) bad |= a.rows[j] == row;
  if (!bad) {
    for (int k = threadIdx.x; k < keep; k += blockDim.x) {
      const int at = a.path[(int64_t)i * a.path_stride + k], before = k ? a.path[(int64_t)i * a.path_stride + k - 1] : -1;
      bad |= at <= before || at >= nn;
    }
    const int p0 = (c - nn) / kPageTokens, kept = pages_of(c - nn + keep);
    for (int p = p0 + threadIdx.x; p < pages_of(c); p += blockDim.x) {
      const int page = a.table[(int64_t)row * a.stride + p];
      if ((unsigned)page >= (unsigned)a.num_pages) bad = true;
      else if (keep < nn && p < kept && a.refs[page] != 1) bad = true;
    }
  }
  return !__syncthreads_or(bad);
}
template <typename W>
__device__ __forceinline__ void accept_column(const AcceptArgs& a, const CacheEntry& ce, uint8_t* base, const int32_t* trow, const int32_t* path, int P, int keep) {
  constexpr int kAhead = 8;                            // loads of as many tokens under way
  auto at = [&](int pos) { return reinterpret_cast<W*>(base + ((int64_t)trow[pos / kPageTokens] * kPageTokens + pos % kPageTokens) * ce.token_bytes); };
  for (int k0 = 0; k0 < keep; k0 += kAhead) {
    W v[kAhead];
    int from[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      from[j] = k0 + j < keep ? path[k0 + j] : -1;
      if (from[j] > k0 + j) v[j] = *at(P + from[j]);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (from[j] > k0 + j) *at(P + k0 + j) = v[j];
  }
}
// The length and the pages of entry i, when all contents have moved; every thread of the CTA has read the length.
__device__ __forceinline__ void accept_pages(const AcceptArgs& a, int row, int c, int now) {
  if (threadIdx.x == 0) a.ctx[row] = now;
  for (int p = pages_of(now) + threadIdx.x; p < pages_of(c); p += blockDim.x) {
    int32_t* entry = a.table + (int64_t)row * a.stride + p;
    const int page = *entry;
    *entry = -1;
    if (atomicSub(&a.refs[page], 1) > 0) continue;
    atomicAdd(&a.refs[page], 1);                       // was free already: the state is not what it says
    if (a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
  }
}
// ALONE: the whole call is one cluster, a CTA a row, and the pages go here: every row has been looked at before one changes.
template <int N, bool ALONE>
__global__ void __launch_bounds__(ALONE ? kAcceptThreads : kCopyThreads) accept_kernel(const AcceptArgs a, const __grid_constant__ AcceptCaches<N> cs, int lead) {
  if (!ALONE) launch_dependents();
  const int i = blockIdx.x, cols = cs.first[cs.n_caches];
  const bool ok = accept_valid(a, i);
  if (ALONE) pool_sync();
  else if (lead && blockIdx.y == 0 && threadIdx.x == 0) a.accepted[i] = ok;
  if (!ok) {
    if (threadIdx.x == 0 && a.status) atomicCAS(a.status, kStatusOk, kStatusBadIndex);
    return;
  }
  const int row = a.rows[i], ctx = a.ctx[row], P = ctx - a.n_new[i], keep = a.n_keep[i];
  const int32_t *trow = a.table + (int64_t)row * a.stride, *path = a.path + (int64_t)i * a.path_stride;
  for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < cols; c += gridDim.y * blockDim.x) {
    int e = 0;
    for (int hi = cs.n_caches; hi - e > 1;) {          // the cache that column c belongs to
      const int mid = (e + hi) / 2;
      (c >= cs.first[mid] ? e : hi) = mid;
    }
    const CacheEntry& ce = cs.cache[e];
    const int wide = ce.token_bytes % 16 == 0 ? 16 : 4, per = ce.token_bytes / wide, in = c - cs.first[e], layer = in / per;
    uint8_t* base = ce.base + layer * ce.layer_stride + (in - layer * per) * wide;
    if (wide == 16) accept_column<uint4>(a, ce, base, trow, path, P, keep);
    else accept_column<uint32_t>(a, ce, base, trow, path, P, keep);
  }
  if (ALONE) {
    __syncthreads();
    accept_pages(a, row, ctx, P + keep);
  }
}
__global__ void __launch_bounds__(kCopyThreads) accept_pages_kernel(const AcceptArgs a) {
  const int i = blockIdx.x;
  if (!grid_wait(a.accepted)[i]) return;
  const int row = a.rows[i], c = a.ctx[row];
  __syncthreads();
  accept_pages(a, row, c, c - a.n_new[i] + a.n_keep[i]);
}

// ---- launches --------------------------------------------------------------------------------------------------------
template <typename... Params, typename... Args>
static void launch_pool(void (*kern)(Params...), int num_pages, size_t smem, cudaStream_t stream, Args... args) {
  // a CTA to every 1024 pages: the plan of compacting 6000 pages takes 12.1 us with one, 9.3 with 2048 pages a CTA, 7.7 so; fewer
  // than 2048 pages do without the cluster's barriers
  const int ctas = min(kPoolCtas, max(1, num_pages / kPoolThreads));
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

// Caches in groups that fit one launch; a.src and what else says which pages is set.  `most`: no more pages than that are copied.  The first
// launch does the other work too, `others` warps of it.
template <int WORK>
static int launch_copies(CopyArgs& a, const PoolArgs& f, const RemapArgs& m, const dsa_page_cache* caches, int n_caches, int64_t most, int64_t others,
                         cudaStream_t stream) {
  int c0 = 0;
  do {
    a.n_caches = min(n_caches - c0, kCopyCaches);
    a.first[0] = 0;
    for (int c = 0; c < a.n_caches; ++c) {
      const dsa_page_cache& h = caches[c0 + c];
      a.cache[c] = {static_cast<uint8_t*>(h.base), h.layer_stride, h.layers, h.token_bytes};
      a.first[c + 1] = a.first[c] + h.layers * ((kPageTokens * h.token_bytes + kCopyChunk - 1) / kCopyChunk);
    }
    const bool lead = WORK != kCopyOnly && c0 == 0;
    const int64_t items = max(most * a.first[a.n_caches], lead ? (others + kCopyThreads / 32 - 2) / (kCopyThreads / 32 - 1) : 0);
    const int grid = (int)min(items, (int64_t)sm_count() * kCopyCtas);
    if (grid > 0) {
      auto kern = lead ? copy_kernel<WORK> : copy_kernel<kCopyOnly>;
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kCopySmem) != cudaSuccess)
        return set_error(DSA_ERR_CUDA, "copy_pages: cannot raise dynamic shared memory to %d", kCopySmem);
      launch_after(lead, kern, dim3(grid), kCopyThreads, kCopySmem, stream, a, f, m);
    }
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
  return launch_copies<kCopyOnly>(a, PoolArgs{}, RemapArgs{}, caches, n_caches, n, 0, stream);
}

static PoolArgs pool_args(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, int n, int32_t* status) {
  PoolArgs a{};
  a.table = table; a.stride = stride; a.P = P; a.B = B;
  a.ctx = ctx; a.refs = refs; a.num_pages = num_pages; a.n = n;
  a.status = status;
  return a;
}

// What the calls that take or move pages need: a few words, and extend the pages taken and two numbers an entry, fork five, compact four
// lists of pages.
size_t pages_workspace_bytes(int num_pages, int n) { return ((size_t)4 * num_pages + (size_t)5 * n + 4) * sizeof(int32_t); }

int extend_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* rows, const int32_t* n_new, int n,
                        int max_new, int32_t* slots, int32_t* workspace, int32_t* status, cudaStream_t stream) {
  PoolArgs a = pool_args(table, stride, P, B, ctx, refs, num_pages, n, status);
  a.a = rows; a.b = n_new;
  a.max_new = max_new;
  a.slots = slots;
  a.refused = workspace;
  a.first = workspace + 4;
  a.held = a.first + n;
  a.fresh = a.held + n;
  const int64_t units = n * extend_per(max_new);
  a.fill = units <= kFillUnits;
  launch_pool(extend_kernel, num_pages, seen_bytes(B), stream, a);
  if (!a.fill) launch_after(1, extend_fill_kernel, dim3((unsigned)min((units + 7) / 8, (int64_t)sm_count() * 8)), 256, 0, stream, a);
  return check_launch("extend_pages");
}

int fork_pages_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* parents, const int32_t* children,
                      int n, const dsa_page_cache* caches, int n_caches, int32_t* workspace, int32_t* status, cudaStream_t stream) {
  PoolArgs a = pool_args(table, stride, P, B, ctx, refs, num_pages, n, status);
  a.a = parents; a.b = children;
  a.refused = workspace;
  a.first = workspace + 4;
  a.fresh = a.first + n;
  a.src = a.fresh + n;
  a.dst = a.src + n;
  a.tokens = a.dst + n;
  launch_pool(fork_kernel, num_pages, seen_bytes(B), stream, a);
  CopyArgs c{};
  c.num_pages = num_pages;
  c.src = a.src; c.dst = a.dst; c.tokens = a.tokens;
  c.n = n;
  c.status = status;
  return launch_copies<kCopyFork>(c, a, RemapArgs{}, caches, n_caches, n, (int64_t)n * max(1, (P + 31) / 32), stream);
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
  c.status = status;
  const RemapArgs m{table, a.remap, a.count, new_table, stride, new_stride, B, P, num_pages};
  return launch_copies<kCopyCompact>(c, PoolArgs{}, m, caches, n_caches, num_pages / 2, ((int64_t)B * P + 31) / 32, stream);
}

// Whether the pages have gone too.
template <int N>
static bool launch_accept(const AcceptArgs& a, const dsa_page_cache* caches, int n_caches, int lead, cudaStream_t stream) {
  AcceptCaches<N> cs;
  cs.n_caches = n_caches;
  cs.first[0] = 0;
  for (int c = 0; c < n_caches; ++c) {
    const dsa_page_cache& h = caches[c];
    cs.cache[c] = {static_cast<uint8_t*>(h.base), h.layer_stride, h.layers, h.token_bytes};
    cs.first[c + 1] = cs.first[c] + h.layers * (h.token_bytes / (h.token_bytes % 16 == 0 ? 16 : 4));
  }
  const int split = min(max(1, (cs.first[n_caches] + kCopyThreads - 1) / kCopyThreads), 65535);
  if constexpr (N == 8) {
    if (a.n <= kAcceptAlone && split * kCopyThreads <= kAcceptThreads) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = a.n;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(a.n);
      cfg.blockDim = dim3(split * kCopyThreads);
      cfg.stream = stream;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      cudaLaunchKernelEx(&cfg, accept_kernel<8, true>, a, cs, lead);      // its error is the launch check's
      return true;
    }
  }
  accept_kernel<N, false><<<dim3(a.n, split), kCopyThreads, 0, stream>>>(a, cs, lead);
  return false;
}

int accept_drafts_launch(int32_t* table, int64_t stride, int P, int B, int32_t* ctx, int32_t* refs, int num_pages, const int32_t* rows, const int32_t* n_new,
                         const int32_t* path, int path_stride, const int32_t* n_keep, int n, const dsa_page_cache* caches, int n_caches, int32_t* workspace,
                         int32_t* status, cudaStream_t stream) {
  AcceptArgs a{};
  a.table = table; a.stride = stride; a.P = P; a.B = B;
  a.ctx = ctx; a.refs = refs; a.num_pages = num_pages; a.n = n;
  a.rows = rows; a.n_new = n_new; a.path = path; a.path_stride = path_stride; a.n_keep = n_keep;
  a.accepted = workspace;
  a.status = status;
  bool done = false;
  if (n_caches <= 8) {
    done = launch_accept<8>(a, caches, n_caches, 1, stream);
  } else {
    for (int c0 = 0; c0 < n_caches; c0 += kCopyCaches) launch_accept<kCopyCaches>(a, caches + c0, min(n_caches - c0, kCopyCaches), c0 == 0, stream);
  }
  if (!done) launch_after(1, accept_pages_kernel, dim3(n), kCopyThreads, 0, stream, a);
  return check_launch("accept_drafts");
}

}  // namespace dsa
