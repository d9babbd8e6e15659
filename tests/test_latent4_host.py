"""The 4-bit record's oracle against its own definition, and what the C entry points refuse before any launch."""
import ctypes
import struct

import numpy as np
import pytest

from llmdivedeep_b200 import _lib, build
from oracle import latent4_oracle as L


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_records_read_back_as_the_values_they_stand_for():
    rng = np.random.default_rng(0)
    kv = rng.standard_normal((40, 576)) * np.exp(rng.standard_normal((40, 1)) * 3)
    kv[0, :16], kv[1, 3], kv[2, 20] = 0, np.inf, np.nan
    kv[3, :16] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -6]
    rope = kv[:, 512:].astype(np.float32)
    kv[:, 512:] = (rope.view(np.uint32) & 0xffff0000).view(np.float32)           # representable in bf16
    bits = np.ascontiguousarray((kv[:, 512:].astype(np.float32).view(np.uint32) >> 16).astype("<u2")).view(np.uint8)
    rec = L.records(kv, bits)
    assert rec.shape == (40, 416)
    np.testing.assert_array_equal(L.decode(rec), L.values(kv))
    assert list(L.values(kv)[3, :16]) == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, -6]
    assert np.isnan(L.values(kv)[1, :16]).all() and np.isnan(L.values(kv)[2, 16:32]).all() and np.isfinite(L.values(kv)[2, :16]).all()
    # nearest: a value is off by at most a sixth of its group's largest (the gap from 4 to 6 halved), and by what the scale is
    ok = np.isfinite(kv[:, :512])
    amax = np.repeat(np.abs(np.where(ok, kv[:, :512], 0)).reshape(-1, 32, 16).max(-1), 16, -1)
    err = np.abs(L.values(kv)[:, :512] - kv[:, :512])
    good = np.isfinite(err)
    assert (err[good] <= (amax / 6 * (1 + 1 / 16) + 2.0 ** -16)[good]).all()
    # and quantising what was read changes nothing
    fine = np.isfinite(L.values(kv)).all(-1)
    np.testing.assert_array_equal(L.values(L.values(kv)[fine]), L.values(kv)[fine])


def test_the_scale_range_ends_where_it_says():
    kv = np.zeros((3, 576))
    kv[0, :16], kv[1, :16], kv[2, 0] = 1e9, 1e-9, 6 * 2.0 ** -15
    v = L.values(kv)
    assert (v[0, :16] == 368640).all() and (v[1, :16] == 0).all() and v[2, 0] == 6 * 2.0 ** -15


def cache_array(*entries):
    return b"".join(struct.pack("=Qqii", *e) for e in entries)


def test_calls_are_refused_with_a_code_and_a_message(lib):
    err = lib.dsa_last_error_string
    # pack / unpack
    assert lib.dsa_pack_latent4(None, 0, 0, 0, None, 0, None, None, None, None, None, None, None) == 0
    assert lib.dsa_pack_latent4(16, 0, 576, -1, 16, 8, 16, None, None, None, None, None, None) == -1
    assert lib.dsa_pack_latent4(None, 0, 576, 4, 16, 8, 16, None, None, None, None, None, None) == -5
    assert lib.dsa_pack_latent4(16, 3, 576, 4, 16, 8, 16, None, None, None, None, None, None) == -5
    assert lib.dsa_pack_latent4(16, 0, 500, 4, 16, 8, 16, None, None, None, None, None, None) == -1
    assert lib.dsa_pack_latent4(16, 0, 577, 4, 16, 8, 16, None, None, None, None, None, None) == -2
    assert lib.dsa_pack_latent4(16, 0, 576, 4, 24, 8, 16, None, None, None, None, None, None) == -2
    assert lib.dsa_pack_latent4(16, 0, 576, 4, 16, 3, None, None, None, None, None, None, None) == -1 and b"in order" in err()
    assert lib.dsa_pack_latent4(16, 0, 576, 4, 16, 8, 16, 16, None, None, None, None, None) == -5
    assert lib.dsa_pack_latent4(16, 0, 576, 4, 16, 8, 16, 8, 16, 16, 16, None, None) == -2
    assert lib.dsa_unpack_latent4(None, 0, None, 0, None, 0, None, None) == 0
    assert lib.dsa_unpack_latent4(16, 3, None, 4, 16, 576, None, None) == -1
    assert lib.dsa_unpack_latent4(16, 64, None, 4, 16, 580, None, None) == -2
    assert lib.dsa_unpack_latent4(16, 64, None, 4, None, 576, None, None) == -5
    # attention
    ok = [16, 16, 416, 16, 1, 1, 16, 16, 1, 16, 64, 1, 64, 0.1, None, 0, None, None]
    for at, bad, code, word in ((2, 400, -1, b"400 bytes"), (5, 0, -1, b"tokens_per_seq"), (10, 4096, -1, b"2048"), (13, -1.0, -5, b"scale"), (1, 8, -2, b"aligned"),
                                (12, 65, -1, b"max_ctx"), (0, None, -5, b"NULL")):
        args = list(ok)
        args[at] = bad
        assert lib.dsa_sparse_mla_decode_records(*args) == code and word in err(), (at, bad, err())
    # pages
    one = cache_array((4096, 0, 1, 416))
    assert lib.dsa_copy_pages(one, 1, 8, None, None, None, 0, None, None) == 0
    assert lib.dsa_copy_pages(one, 1, 8, None, 16, None, 2, None, None) == -5
    assert lib.dsa_copy_pages(None, 1, 8, 16, 16, None, 2, None, None) == -5
    assert lib.dsa_copy_pages(one, 1, -8, 16, 16, None, 2, None, None) == -1
    assert lib.dsa_copy_pages(cache_array((4096, 0, 1, 6)), 1, 8, 16, 16, None, 2, None, None) == -1
    assert lib.dsa_copy_pages(cache_array((4100, 0, 1, 8)), 1, 8, 16, 16, None, 2, None, None) == -2
    assert lib.dsa_copy_pages(cache_array((4096, 8, 2, 8)), 1, 8, 16, 16, None, 2, None, None) == -2
    big = lib.dsa_pages_workspace_bytes(8, 2)
    assert big >= (4 * 8 + 5 * 2) * 4 and lib.dsa_pages_workspace_bytes(-1, 2) == 0
    ext = [16, 4, 4, 3, 16, 16, 8, 16, 16, 2, 5, 16, 16, big, None, None]
    for at, bad, code in ((1, 3, -1), (2, -1, -1), (3, 1 << 19, -1), (6, 1 << 26, -1), (10, -1, -1), (4, None, -5), (7, None, -5), (11, None, -5), (12, None, -3),
                          (13, big - 1, -3), (12, 18, -3)):
        args = list(ext)
        args[at] = bad
        assert lib.dsa_extend_pages(*args) == code, (at, bad, err())
    args = list(ext)
    args[9] = 0
    assert lib.dsa_extend_pages(*args) == 0                        # nothing asked for
    fork = [16, 4, 4, 3, 16, 16, 8, 16, 16, 2, one, 1, 16, big, None, None]
    for at, bad, code in ((1, 3, -1), (7, None, -5), (8, None, -5), (10, None, -5), (11, -1, -1), (12, None, -3), (13, big - 1, -3)):
        args = list(fork)
        args[at] = bad
        assert lib.dsa_fork_pages(*args) == code, (at, bad, err())
    assert lib.dsa_free_pages(16, 4, 4, 3, None, 16, 8, 16, 2, None, None) == -5
    assert lib.dsa_free_pages(16, 4, 4, 3, 16, 16, 8, None, 2, None, None) == -5
    assert lib.dsa_free_pages(None, 4, 4, 3, 16, 16, 8, None, 0, None, None) == -5
    assert lib.dsa_compact_pages(16, 4, 16, 3, 4, 3, 16, 16, 8, one, 1, 16, big, None, None) == -1
    assert lib.dsa_compact_pages(16, 4, 16, 4, 4, 3, 16, None, 8, one, 1, 16, big, None, None) == -5
    assert lib.dsa_compact_pages(16, 4, 16, 4, 4, 3, 16, 16, 8, one, 1, None, big, None, None) == -3


def test_page_cache_struct_is_what_the_binding_packs():
    class C(ctypes.Structure):
        _fields_ = [("base", ctypes.c_void_p), ("layer_stride", ctypes.c_int64), ("layers", ctypes.c_int32), ("token_bytes", ctypes.c_int32)]

    c = C.from_buffer_copy(cache_array((4096, 77, 3, 416)))
    assert ctypes.sizeof(C) == 24 and (c.base, c.layer_stride, c.layers, c.token_bytes) == (4096, 77, 3, 416)


def test_pool_oracle_keeps_its_own_rules():
    """References equal the holders after every step, and a sequence's contents survive forks, frees and compactions."""
    rng = np.random.default_rng(5)
    B, P, pages = 7, 5, 26
    pool = L.Pool(np.full((B, P), -1, np.int32), np.zeros(B, np.int32), np.zeros(pages, np.int32), [np.zeros((2, pages * 64, 1), np.int64)])
    text = [[] for _ in range(B)]
    for step in range(400):
        kind = rng.integers(4)
        r = rng.permutation(B)
        if kind == 0:
            n_new = rng.integers(0, 100, 2)
            slots = pool.extend(r[:2], n_new, 100)
            for row, s in zip(r[:2], slots):
                new = rng.integers(1, 1 << 40, (s >= 0).sum())
                text[row] += list(new)
                for c in pool.caches:
                    c[:, s[s >= 0], 0] = new
        elif kind == 1:
            before = pool.status
            pool.status = 0
            pool.fork(r[:2], r[2:4])
            if pool.status == 0:
                for p, c in zip(r[:2], r[2:4]):
                    text[c] = list(text[p])
            pool.status = before
        elif kind == 2:
            pool.free(r[:2])
            text[r[0]], text[r[1]] = [], []
        else:
            pool.compact()
            assert (pool.refs[:(pool.refs > 0).sum()] > 0).all()
        held = np.zeros(pages, int)
        for row in range(B):
            n = len(text[row])
            assert pool.ctx[row] == n
            pos = np.arange(n)
            assert (pool.caches[0][1, pool.table[row][pos // 64] * 64 + pos % 64, 0] == text[row]).all()
            np.add.at(held, pool.table[row][pool.table[row] >= 0], 1)
        assert (held == pool.refs).all()
