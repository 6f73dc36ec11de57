"""The token-major operators without a GPU: how packed sequences are cut into tiles, and what the C entry points refuse."""
import ctypes
import os

import numpy as np
import pytest

from tests.conftest import ROOT


def _tiles(q_len, k_len, rows_per_token, rows_per_tile, lead=0, behind=0):
    from visual_odometry_amd.build import build_host_checks
    lib = ctypes.CDLL(build_host_checks())
    fn = lib.host_row_tiles
    fn.restype = ctypes.c_int64
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    q = np.concatenate([[lead], lead + np.cumsum(q_len)]).astype(np.int32)
    k = np.concatenate([[0], np.cumsum(k_len)]).astype(np.int32)
    args = (q.ctypes.data, k.ctypes.data, len(q_len), int(q[-1]) + behind, int(k[-1]), rows_per_token, rows_per_tile)
    n = fn(*args, None)
    out = np.zeros((n, 6), np.int64)
    fn(*args, out.ctypes.data)
    return q, k, out


@pytest.mark.parametrize("rows_per_token,rows_per_tile", [(1, 128), (1, 32), (4, 32), (8, 32), (7, 32), (40, 32), (1, 1)])
@pytest.mark.parametrize("seed", range(12))
def test_every_row_of_every_sequence_lies_in_exactly_one_tile(rows_per_token, rows_per_tile, seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 40))
    q_len = rng.integers(0, [2, 40, 300][seed % 3], n)
    if seed % 4 == 0:
        q_len[rng.integers(0, n, n // 2)] = 0
    k_len = rng.integers(0, 50, n)
    q, k, tiles = _tiles(q_len, k_len, rows_per_token, rows_per_tile, lead=int(rng.integers(0, 300)) if seed % 2 else 0, behind=seed * 7)
    hits = [np.zeros(l * rows_per_token, int) for l in q_len]
    for any_, row, q0, Lq, k0, Lk in tiles:
        if not any_:
            continue
        s = int(np.flatnonzero((q[:-1] == q0) & (q_len == Lq) & (k[:-1] == k0) & (k_len == Lk))[0])
        assert row % rows_per_tile == 0
        hits[s][row:row + rows_per_tile] += 1
    # sequences that are alike in all four numbers are empty ones
    for s, h in enumerate(hits):
        assert (h == 1).all(), (s, q_len)


def test_wrong_offsets_never_lead_outside_the_tensors():
    from visual_odometry_amd.build import build_host_checks
    lib = ctypes.CDLL(build_host_checks())
    lib.host_row_tiles.restype = ctypes.c_int64
    rng = np.random.default_rng(0)
    for _ in range(50):
        S, Tq, Tk = int(rng.integers(1, 9)), int(rng.integers(1, 500)), int(rng.integers(0, 500))
        q = rng.integers(-2 ** 31, 2 ** 31, S + 1).astype(np.int32) if rng.random() < 0.5 else rng.integers(-50, 700, S + 1).astype(np.int32)
        k = rng.integers(-50, 700, S + 1).astype(np.int32)
        out = np.zeros((Tq // 32 + S, 6), np.int64)
        n = lib.host_row_tiles(q.ctypes.data_as(ctypes.c_void_p), k.ctypes.data_as(ctypes.c_void_p), S, ctypes.c_int64(Tq), ctypes.c_int64(Tk),
                               1, 32, out.ctypes.data_as(ctypes.c_void_p))
        assert n == len(out)
        for any_, row, q0, Lq, k0, Lk in out:
            assert 0 <= q0 and 0 <= Lq and q0 + Lq <= Tq and 0 <= k0 and 0 <= Lk and k0 + Lk <= Tk
            assert not any_ or 0 <= row < Lq


@pytest.mark.parametrize("sequences", [62, 63, 64, 65, 66, 127, 500, 5000])
@pytest.mark.parametrize("shape", ["equal", "rising", "one_long", "empty_but_for_some"])
def test_tiles_of_many_sequences(sequences, shape):
    """Lengths for which a sequence lies where equal ones would put it, and lengths for which it does not."""
    q_len = {"equal": np.full(sequences, 40), "rising": np.arange(sequences) % 700 // 3, "one_long": np.full(sequences, 1),
             "empty_but_for_some": np.arange(sequences) % 50 // 49 * 130}[shape].copy()
    if shape == "one_long":
        q_len[sequences // 3] = 20000
    k_len = np.arange(sequences) % 7                                  # tells neighbours apart
    q, k, tiles = _tiles(q_len, k_len, 1, 32, lead=5)
    hits = [0] * sequences
    for any_, row, q0, Lq, k0, Lk in tiles:
        if any_:
            s = int(np.flatnonzero((q[:-1] == q0) & (q_len == Lq) & (k[:-1] == k0) & (k_len == Lk))[0])
            assert row == 32 * hits[s]
            hits[s] += 1
    assert hits == [-(-int(l) // 32) for l in q_len]


def test_linear_entry_point_refuses():
    from visual_odometry_amd import _lib
    lib = _lib.load()
    p = ctypes.cast((ctypes.c_char * 4096)(), ctypes.c_void_p)

    def call(x=p, xs=16, w=p, b=None, r=None, rs=0, y=p, ys=8, M=4, C=16, K=8, act=0, dt=1, ws=None, wb=0):
        return lib.vo_linear(x, xs, w, b, r, rs, y, ys, M, C, K, act, dt, ws, wb, None)
    for kw in (dict(dt=3), dict(dt=-1), dict(act=5), dict(act=-1), dict(M=-1), dict(C=0), dict(K=0), dict(x=None), dict(w=None), dict(y=None),
               dict(xs=15), dict(ys=7), dict(r=p, rs=7)):
        assert call(**kw) == _lib.VO_ERR_INVALID_ARG, kw
        assert lib.vo_last_error()
    assert call(M=0) == _lib.VO_OK                                                  # nothing to do, nothing launched
    assert call(xs=1 << 22) == _lib.VO_ERR_UNSUPPORTED and call(xs=1 << 23, C=1 << 23) == _lib.VO_ERR_UNSUPPORTED
    # more threads than a launch has
    assert call(M=1 << 32, C=8, K=8) == _lib.VO_ERR_UNSUPPORTED and b"too large" in lib.vo_last_error()
    assert call(M=1, C=8, K=(1 << 31) - 1, ys=1 << 31) == _lib.VO_ERR_UNSUPPORTED and b"too large" in lib.vo_last_error()
    # a shape that is split over C needs its workspace
    need = lib.vo_linear_workspace_bytes(1, 65536, 16, _lib.VO_PIECES_F16)
    assert need > 0
    big = dict(M=1, C=65536, K=16, xs=65536, ys=16)
    assert call(**big) == _lib.VO_ERR_INVALID_ARG and b"workspace" in lib.vo_last_error()
    assert call(**big, ws=p, wb=need - 1) == _lib.VO_ERR_INVALID_ARG
    assert call(**big, ws=ctypes.c_void_p(p.value + 4), wb=need) == _lib.VO_ERR_INVALID_ARG
    assert lib.vo_linear_workspace_bytes(0, 16, 16, 0) == 0 and lib.vo_linear_workspace_bytes(-5, 16, 16, 0) == 0


def test_attention_entry_point_refuses():
    from visual_odometry_amd import _lib
    lib = _lib.load()
    p = ctypes.cast((ctypes.c_char * 4096)(), ctypes.c_void_p)
    p = ctypes.c_void_p((p.value + 15) // 16 * 16)

    def call(q=p, qs=64, qh=32, k=p, ks=64, kh=32, v=p, vs=64, vh=32, o=p, os=64, oh=32, qo=None, ko=None, S=1, Tq=4, Tk=4, Hq=2, Hk=2, D=32,
             scale=1.0, causal=0, dt=1, ws=None, wb=0):
        return lib.vo_attention(q, qs, qh, k, ks, kh, v, vs, vh, o, os, oh, qo, ko, S, Tq, Tk, Hq, Hk, D, scale, causal, dt, ws, wb, None)
    for kw in (dict(dt=3), dict(S=0), dict(Tq=-1), dict(Tk=-1), dict(Hq=0), dict(Hk=0), dict(Hq=3), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(S=2), dict(qo=p), dict(ko=p), dict(q=None), dict(k=None), dict(v=None), dict(o=None)):
        assert call(**kw) == _lib.VO_ERR_INVALID_ARG, kw
        assert lib.vo_last_error()
    for kw in (dict(D=0), dict(D=264), dict(D=12), dict(qs=60), dict(kh=4), dict(vs=-64), dict(os=1 << 23), dict(q=ctypes.c_void_p(p.value + 8)),
               dict(o=ctypes.c_void_p(p.value + 2)), dict(Tq=1 << 31), dict(Tk=1 << 31), dict(dt=0, D=30)):
        assert call(**kw) == _lib.VO_ERR_UNSUPPORTED, kw
    assert call(Tq=(1 << 31) - 1, Hq=64, Hk=64) == _lib.VO_ERR_UNSUPPORTED and b"too many" in lib.vo_last_error()
    assert call(scale=1e-38) == _lib.VO_ERR_INVALID_ARG and call(scale=1e38) == _lib.VO_ERR_INVALID_ARG
    assert call(Tq=0) == _lib.VO_OK
    need = lib.vo_attention_workspace_bytes(1, 65536, 1, 2, 2, 32, 1)
    assert need > 0 and call(Tq=1, Tk=65536) == _lib.VO_ERR_INVALID_ARG and b"workspace" in lib.vo_last_error()
    assert call(Tq=1, Tk=65536, ws=p, wb=need - 1) == _lib.VO_ERR_INVALID_ARG
    assert lib.vo_attention_workspace_bytes(1, 65536, 1, 3, 2, 32, 1) == 0 and lib.vo_attention_workspace_bytes(0, 5, 1, 2, 2, 32, 1) == 0


def test_the_python_entry_points_refuse_cpu_tensors():
    import torch
    from visual_odometry_amd import ops
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.linear(torch.zeros(2, 8), torch.zeros(4, 8))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.attention(torch.zeros(2, 1, 8), torch.zeros(2, 1, 8), torch.zeros(2, 1, 8))


def test_overlaps_are_found_and_column_ranges_are_none():
    """Against the elements themselves: two random strided views of one buffer that share an element are always refused, and rows the same
    distance apart never where they share no column."""
    import random
    import torch
    from visual_odometry_amd import ops
    rng, base, ids = random.Random(0), torch.zeros(2000, dtype=torch.float16), torch.arange(2000)

    def view(step=0):
        if step or rng.random() < 0.6:
            n = (rng.randint(2 if step else 1, 6), rng.randint(1, 12))
            return n, (step or rng.choice([n[1], n[1] + rng.randint(0, 30), 48, 24]), 1), rng.randint(0, 200)
        n = (rng.randint(1, 5), rng.randint(1, 3), rng.randint(1, 8))
        return n, rng.choice([(n[1] * n[2] + rng.randint(0, 30), n[2], 1), (48, n[2] + rng.randint(0, 4), 1),
                              (n[2], n[0] * n[2] + rng.randint(0, 9), 1), (96, 0, 1)]), rng.randint(0, 200)

    def refused(a, b):
        try:
            ops._no_overlap(a, b, "x")
        except ValueError:
            return True
        return False
    for step in [0] * 3000 + [40] * 3000:
        a, b = view(step), view(step)
        shared = bool(set(ids.as_strided(*a).flatten().tolist()) & set(ids.as_strided(*b).flatten().tolist()))
        says = refused(base.as_strided(*a), base.as_strided(*b))
        assert says or not shared, (a, b)
        if step:
            columns = [{(v[2] + i) % step for i in range(v[0][1])} for v in (a, b)]
            assert not says or columns[0] & columns[1], (a, b)


def test_more_threads_than_a_launch_has_are_refused_also_where_the_count_passes_64_bits():
    from visual_odometry_amd import _lib
    lib = _lib.load()
    p = ctypes.cast((ctypes.c_char * 4096)(), ctypes.c_void_p)
    p = ctypes.c_void_p((p.value + 15) // 16 * 16)

    def attention(S, T, H, D=32, dt=1):
        return lib.vo_attention(p, H * D, D, p, H * D, D, p, H * D, D, p, H * D, D, p, p, S, T, T, H, H, D, 1.0, 0, dt, p, 1 << 60, None)

    def linear(M, C, K):
        return lib.vo_linear(p, C, p, None, None, 0, p, K, M, C, K, 0, 1, p, 1 << 60, None)
    # ten million single tokens: as many workgroups of up to 512 threads
    for D, dt in ((32, 1), (128, 2), (32, 0), (64, 0)):
        assert attention(10_000_000, 10_000_000, 1, D, dt) == _lib.VO_ERR_UNSUPPORTED and b"too many" in lib.vo_last_error()
    big = (1 << 31) - 1
    assert lib.vo_attention(p, 0, 0, p, 0, 0, p, 0, 0, p, 32, 0, p, p, big, 1, 1, big, big, 32, 1.0, 0, 1, p, 1 << 60, None) == _lib.VO_ERR_UNSUPPORTED
    assert lib.vo_attention_workspace_bytes(1, 1, big, big, big, 32, 1) == 0
    for M, K in ((1 << 55, 1 << 17), (1 << 62, 1 << 20), ((1 << 63) - 1, 64), (1 << 45, 1 << 30)):
        assert linear(M, 8, K) == _lib.VO_ERR_UNSUPPORTED and b"too large" in lib.vo_last_error(), (M, K)
        assert lib.vo_linear_workspace_bytes(M, 8, K, 1) == 0
