"""ops.attention against the definition in float64, element by element.

Tolerance, derived.  With A = sum_j p_j |v_j| (p the exact weights):
  * a score is off by at most 2 (D+2) 2^-24 scale sum |q||k| (any order, doubled for truncating additions inside the matrix
    instruction), the exponent's argument by a few more roundings of |s| and |m|, the exponential by 2^-21 of itself: the
    weight's relative error eta, which enters the numerator and the denominator once each;
  * with 16-bit storage the weight is rounded once, by eps / 2 of itself (float16: by 2^-25 at least, of weights whose
    largest is at least 1, so 2^-25 sum |v| / l more, l >= 1);
  * the two sums over n keys are float32: 2 (n + 64) 2^-24 of A each, and one rescaling per key tile;
  * the store rounds once, by eps / 2 of the value."""
import numpy as np
import pytest
import torch

from visual_odometry_amd import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U32 = 2.0 ** -24


def reference(q, k, v, q_len, k_len, causal, scale):
    """(out, tolerance) in float64 for packed sequences."""
    dt, D, Hq, Hk = q.dtype, q.shape[2], q.shape[1], k.shape[1]
    half = torch.finfo(dt).eps / 2
    out = torch.zeros(sum(q_len), Hq, D, device=q.device, dtype=torch.float64)
    tol = torch.zeros_like(out)
    a = b = 0
    for lq, lk in zip(q_len, k_len):
        for h in range(Hq):
            if lq == 0 or lk == 0:
                continue
            Q, K, V = q[a:a + lq, h].double(), k[b:b + lk, h // (Hq // Hk)].double(), v[b:b + lk, h // (Hq // Hk)].double()
            S = Q @ K.t().contiguous() * scale
            B = Q.abs() @ K.abs().t().contiguous() * scale
            see = torch.ones(lq, lk, device=q.device, dtype=torch.bool)
            if causal:
                see = see.tril(lk - lq)
            S = S.masked_fill(~see, -torch.inf)
            some = see.any(1)
            m = torch.where(some, S.amax(1), torch.zeros_like(S[:, 0]))
            e = torch.exp(S - m[:, None])
            l = e.sum(1)
            p = e / torch.where(some, l, torch.ones_like(l))[:, None]
            o, A = p @ V, p @ V.abs()
            x = 2 * (D + 2) * U32 * B + 4 * U32 * (torch.where(see, S, torch.zeros_like(S)).abs() + m.abs()[:, None] + 8)
            eta = (torch.where(see, torch.expm1(x), torch.zeros_like(x)).amax(1) + 2.0 ** -21)[:, None]
            rnd = 0.0 if dt == torch.float32 else half
            t = A * (2 * eta + rnd + 4 * (lk + 64) * U32) * 1.05
            if dt == torch.float16:
                t = t + 2.0 ** -25 * (see.double() @ V.abs()) / torch.where(some, l, torch.ones_like(l))[:, None]
            t = t + half * (o.abs() + t) + {torch.float32: 2.0 ** -120, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -120}.get(dt, 0.0)
            out[a:a + lq, h], tol[a:a + lq, h] = o, t
        a, b = a + lq, b + lk
    return out, tol


def offsets(lengths, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(lengths)]).astype(np.int32)).cuda()


def make(q_len, k_len, Hq, Hk, D, dtype, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return ((n(sum(q_len), Hq, D) * spread).to(dtype), n(sum(k_len), Hk, D).to(dtype), n(sum(k_len), Hk, D).to(dtype))


def check(y, want, tol):
    assert y.shape == want.shape
    err = (y.double() - want).abs()
    assert bool((err <= tol).all()), f"error {(err / tol).nan_to_num(0).max().item():.3g} times the bound"


def run(q_len, k_len, Hq, Hk, D, dtype, causal, seed=0, scale=None, spread=1.0):
    q, k, v = make(q_len, k_len, Hq, Hk, D, dtype, seed, spread)
    y = ops.attention(q, k, v, offsets(q_len), offsets(k_len), causal=causal, scale=scale)
    assert y.dtype == dtype
    check(y, *reference(q, k, v, q_len, k_len, causal, D ** -0.5 if scale is None else scale))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 64, 72, 96, 128, 200, 256])
@pytest.mark.parametrize("form", ["tiles", "rows"])
def test_head_sizes(vo, dtype, causal, D, form):
    if form == "tiles":
        run([130, 1, 0, 67], [130, 1, 5, 200], 4, 2, D, dtype, causal, D)
    else:
        run([1, 3, 0, 1], [70, 140, 5, 1], 4, 2, D, dtype, causal, D)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len,k_len", [
    ([1], [1]), ([1], [31]), ([1], [32]), ([1], [33]), ([2], [64]), ([5], [65]), ([33], [127]), ([127], [128]), ([128], [128]), ([129], [129]),
    ([255], [257]), ([300], [64]), ([64], [0]), ([0], [64]), ([0, 0, 7], [3, 0, 9]),
    ([40, 0, 1, 128, 3], [20, 7, 0, 100, 5]),                          # more rows than keys: causal leaves rows empty
    ([160] * 12, [160] * 12), ([1] * 50, list(range(50))), ([513, 2, 90], [700, 1000, 90])])
@pytest.mark.parametrize("Hq,Hk", [(3, 3), (8, 2)])
def test_lengths(vo, dtype, causal, q_len, k_len, Hq, Hk):
    run(q_len, k_len, Hq, Hk, 64, dtype, causal, len(q_len) + sum(q_len))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (32, 8), (40, 1), (6, 3), (128, 1), (129, 1), (260, 2)])
@pytest.mark.parametrize("q_len,k_len", [([1, 1, 1], [700, 3, 90]), ([4, 2, 7], [300, 2, 50]), ([150], [150])])
def test_groups_of_heads(vo, dtype, Hq, Hk, q_len, k_len):
    run(q_len, k_len, Hq, Hk, 32, dtype, True, Hq)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len,k_len,Hq,Hk,D", [
    ([1], [5003], 4, 1, 128), ([1, 2, 1], [4000, 1, 9001], 8, 2, 64), ([3], [2500], 2, 1, 256),       # rows, split over the keys
    ([1], [5003], 4, 1, 96), ([100], [6007], 2, 1, 72),
    ([100], [6007], 2, 1, 64), ([40, 70], [3000, 2500], 2, 2, 128), ([129], [1500], 1, 1, 256)])      # tiles, split over the keys
def test_long_axes_are_split_and_joined(vo, dtype, causal, q_len, k_len, Hq, Hk, D):
    from visual_odometry_amd import _lib
    assert _lib.load().vo_attention_workspace_bytes(sum(q_len), sum(k_len), len(q_len), Hq, Hk, D, ops._TOKEN_DTYPES[dtype]) > 0
    run(q_len, k_len, Hq, Hk, D, dtype, causal, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [([140], [300]), ([2], [300]), ([1], [4000])])
def test_large_scores_and_other_scales(vo, dtype, q_len, k_len):
    """Scores of some hundreds: the maximum moves from tile to tile and nearly all weight lies on a few keys."""
    run(q_len, k_len, 2, 2, 64, dtype, False, 3, spread=12.0)
    run(q_len, k_len, 2, 2, 64, dtype, True, 4, scale=0.01)
    run(q_len, k_len, 2, 2, 64, dtype, True, 4, scale=3.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len", [[130], [2]])
def test_rising_and_falling_scores(vo, dtype, q_len):
    """Keys whose scores rise by a little less or more than the rescaling threshold from tile to tile, or only fall."""
    n, D = 640, 32
    for slope in (0.02, 0.05, 0.1, 0.5, -0.1):
        q, k, v = make(q_len, [n], 1, 1, D, dtype, 9)
        q = torch.zeros_like(q); q[..., 0] = 1
        k = k * 0.01; k[:, 0, 0] = (torch.arange(n, device="cuda") * slope - 20).to(dtype)
        y = ops.attention(q, k, v, scale=1.0)
        check(y, *reference(q, k, v, q_len, [n], False, 1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [[150, 33, 0, 260], [1, 2, 1]])
def test_slices_of_one_projection_and_a_strided_result(vo, dtype, causal, lens):
    Hq, Hk, D = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(sum(lens), (Hq + 2 * Hk + 1) * D, generator=g, device="cuda").to(dtype).view(sum(lens), -1, D)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:Hq + 2 * Hk]
    hold = torch.full((sum(lens), 2 * Hq, 2 * D), 7.0, device="cuda", dtype=dtype)
    out = hold[:, ::2, D:]
    y = ops.attention(q, k, v, offsets(lens), causal=causal, out=out)
    assert y is out
    check(out, *reference(q, k, v, lens, lens, causal, D ** -0.5))
    y = y.clone()
    hold[:, ::2, D:] = 7
    assert bool((hold == 7).all())
    # heads ahead of tokens in memory
    qt, kt, vt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    assert torch.equal(ops.attention(qt, kt, vt, offsets(lens), causal=causal), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len,k_len", [([140, 3, 60], [200, 70, 60]), ([1, 2, 1], [77, 5, 130]), ([1, 1], [2500, 1300])])
def test_what_lies_outside_every_sequence_neither_matters_nor_changes(vo, dtype, causal, q_len, k_len):
    """Rows and keys ahead of the first and behind the last sequence (a padded batch, a cache's unused end) are NaN."""
    lead, behind, D = 5, 140, 64
    q, k, v = make(q_len, k_len, 4, 2, D, dtype, 8)
    pad = lambda t: torch.nn.functional.pad(t.transpose(0, 2), (lead, behind), value=float("nan")).transpose(0, 2).contiguous()
    out = torch.full((lead + sum(q_len) + behind, 4, D), 7.0, device="cuda", dtype=dtype)
    ops.attention(pad(q), pad(k), pad(v), offsets(q_len, lead), offsets(k_len, lead), causal=causal, out=out)
    check(out[lead:lead + sum(q_len)], *reference(q, k, v, q_len, k_len, causal, D ** -0.5))
    assert bool((out[:lead] == 7).all()) and bool((out[lead + sum(q_len):] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [([140, 3], [200, 70]), ([1, 2], [77, 50])])
def test_sequences_do_not_disturb_each_other(vo, dtype, q_len, k_len):
    """NaN and infinity in one sequence stay in it, whatever shares its tiles of memory."""
    q, k, v = make(q_len, k_len, 2, 1, 64, dtype, 6)
    k[k_len[0] - 1] = float("inf"); v[k_len[0] - 2] = float("nan")
    y = ops.attention(q, k, v, offsets(q_len), offsets(k_len))
    assert bool(y[:q_len[0]].isnan().all())
    want, tol = reference(q[q_len[0]:], k[k_len[0]:], v[k_len[0]:], q_len[1:], k_len[1:], False, 0.125)
    check(y[q_len[0]:], want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("q_len,k_len", [([200], [200]), ([130], [300]), ([100], [60]), ([5], [90]), ([3], [2000]), ([140], [2000])])
def test_unbounded_keys_and_values_reach_only_the_rows_that_see_them(vo, dtype, D, q_len, k_len):
    """Causal, with an infinity in one value, a NaN in another key and value near the diagonal: rows ahead of them are exact,
    rows that see them have them."""
    lq, lk = q_len[0], k_len[0]
    q, k, v = make(q_len, k_len, 2, 1, D, dtype, 7)
    clean = reference(q, k, v, q_len, k_len, True, D ** -0.5)
    first = max(lk - lq // 2, lk - 90, 1)                              # a key that the later half of the rows sees
    v[first, 0, 1] = float("inf")
    for name, at in (("value", None), ("key", min(first + 7, lk - 1))):
        if at is not None:
            k[at, 0, 0] = float("nan")
            v[at, 0, D - 1] = float("nan")
        y = ops.attention(q, k, v, causal=True)
        sees = torch.arange(lq, device="cuda") + lk - lq
        ahead = sees < first
        err = (y.double() - clean[0]).abs()
        assert bool((err[ahead] <= clean[1][ahead]).all())
        assert bool((y[~ahead][:, :, 1] == float("inf")).all()) or at is not None
        others = [j for j in range(D) if j != 1]
        if at is None:
            assert bool((err[~ahead][:, :, others] <= clean[1][~ahead][:, :, others]).all())
        else:
            assert bool(y[sees >= at].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [([200], [200]), ([140], [4000]), ([3], [90]), ([3], [4000])])
def test_a_row_of_nan_stays_nan(vo, dtype, q_len, k_len):
    """A query that is not a number has no result, also where its keys are cut into parts; its neighbours do not notice."""
    q, k, v = make(q_len, k_len, 2, 1, 64, dtype, 11)
    want, tol = reference(q, k, v, q_len, k_len, False, 0.125)
    q[1, 1, 5] = float("nan")
    y = ops.attention(q, k, v)
    assert bool(y[1, 1].isnan().all())
    want[1, 1] = tol[1, 1] = 0
    y[1, 1] = 0
    check(y, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("q_len,k_len", [([140], [140]), ([140], [4000]), ([3], [90]), ([3], [4000])])
def test_nan_among_keys_of_no_weight_is_not_lost(vo, dtype, what, q_len, k_len):
    """The first keys' weights underflow to zero beside the last key's, a NaN among them (in a part of their own, where the keys
    are cut) still reaches every row that sees it."""
    q, k, v = make(q_len, k_len, 1, 1, 64, dtype, 12)
    q[:], k[:], k[-1] = 8.0, -1.0, 8.0                                # scores -64 and 512: e^-576 is no float32
    (k if what == "key" else v)[2, 0] = float("nan")
    assert bool(ops.attention(q, k, v).isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_offsets_everything_is_one_sequence(vo, dtype):
    q, k, v = make([200], [333], 4, 4, 64, dtype, 1)
    assert torch.equal(ops.attention(q, k, v, causal=True), ops.attention(q, k, v, offsets([200]), offsets([333]), causal=True))
    assert tuple(ops.attention(q[:0], k, v).shape) == (0, 4, 64)
    assert bool((ops.attention(q, k[:0], v[:0]) == 0).all())


@pytest.mark.parametrize("q_len,k_len", [([200, 40], [200, 40]), ([1, 1], [3000, 40]), ([60], [3000])])
def test_equal_bits_on_another_stream_and_in_a_graph(vo, q_len, k_len):
    q, k, v = make(q_len, k_len, 4, 2, 64, torch.bfloat16, 1)
    qo, ko = offsets(q_len), offsets(k_len)
    want = ops.attention(q, k, v, qo, ko, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [ops.attention(q, k, v, qo, ko, causal=True) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(y, want) for y in ys)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.attention(q, k, v, qo, ko, causal=True)
    for seed in range(4):                                            # new values and new lengths in the same buffers
        for t, n in zip((q, k, v), make(q_len, k_len, 4, 2, 64, torch.bfloat16, 20 + seed)):
            t.copy_(n)
        if len(k_len) > 1:
            ko.copy_(offsets([k_len[0] - seed * 17, k_len[1] + seed * 17]))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.attention(q, k, v, qo, ko, causal=True))


def test_two_streams_at_once(vo):
    """Calls that need workspaces, under way on two streams together."""
    for q_len, k_len in (([1, 1], [5000, 3000]), ([60], [3000])):
        sets = [make(q_len, k_len, 4, 2, 64, torch.bfloat16, 30 + i) for i in range(2)]
        qo, ko = offsets(q_len), offsets(k_len)
        want = [ops.attention(q, k, v, qo, ko, causal=True) for q, k, v in sets]
        streams = [torch.cuda.Stream() for _ in sets]
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for _ in range(20):
            for i, (st, (q, k, v)) in enumerate(zip(streams, sets)):
                with torch.cuda.stream(st):
                    got[i].append(ops.attention(q, k, v, qo, ko, causal=True))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len", [[40], [2]])
def test_four_features_and_shared_heads_by_stride(vo, causal, q_len):
    """The smallest float32 head, and key heads that are one head repeated by a stride of zero."""
    q, k, v = make(q_len, [70], 6, 1, 4, torch.float32, 3)
    y = ops.attention(q, k, v, causal=causal)
    check(y, *reference(q, k, v, q_len, [70], causal, 0.5))
    check(ops.attention(q, k.expand(70, 6, 4), v.expand(70, 6, 4), causal=causal), *reference(q, k, v, q_len, [70], causal, 0.5))


def test_more_sequences_than_a_wave_tests_at_once(vo):
    """Hundreds and thousands of sequences, empty ones and single tokens among them, in both forms."""
    rng = np.random.default_rng(4)
    for n, top in ((65, 3), (700, 2), (4500, 2), (130, 40)):
        q_len = rng.integers(0, top + 1, n).tolist()
        k_len = [int(x) for x in rng.integers(0, 9, n)]
        q, k, v = make(q_len, k_len, 1, 1, 32, torch.float16, n)
        y = ops.attention(q, k, v, offsets(q_len), offsets(k_len))
        seq = np.repeat(np.arange(n), q_len)
        pos = torch.tensor(np.repeat(np.arange(n), k_len)).cuda()
        S = (q[:, 0].double() @ k[:, 0].double().t().contiguous()) * 32 ** -0.5
        S = S.masked_fill(torch.tensor(seq).cuda()[:, None] != pos[None, :], -torch.inf)
        P = torch.softmax(S, 1).nan_to_num(0)
        want = P @ v[:, 0].double()
        # a handful of keys a row: the weights' and the result's roundings, 2^-11 each of sum p |v| (<= 5 here), dominate
        assert float((y[:, 0].double() - want).abs().max()) < 2 * 5 * 2.0 ** -11 * 1.1


def test_a_long_cache_passes_32_bit_offsets(vo):
    """Keys and values more than 2^31 elements (and 2^32 bytes) apart: a cache of 70000 tokens at a stride of 32768."""
    n, D, stride = 70000, 64, 32768
    hold = torch.zeros(n * stride, device="cuda", dtype=torch.float16)
    kv = hold.view(n, stride // D, D)[:, :2]
    g = torch.Generator(device="cuda").manual_seed(3)
    kv.copy_(torch.randn(n, 2, D, generator=g, device="cuda"))
    for lq in (1, 130):
        q = torch.randn(lq, 1, D, generator=g, device="cuda").half()
        y = ops.attention(q, kv[:, :1], kv[:, 1:], causal=True)
        check(y, *reference(q, kv[:, :1], kv[:, 1:], [lq], [n], True, D ** -0.5))


def test_a_block_of_projections_around_attention(vo):
    """As they are used together: fused projection, attention on its slices, projection back onto the residual, perceptron."""
    lens, Hq, Hk, D, W = [160, 33, 160, 7], 4, 2, 64, 256
    T = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    for dtype, tol in ((torch.float32, 2e-5), (torch.float16, 2e-2), (torch.bfloat16, 1.5e-1)):
        x = n(T, W).to(dtype)
        ws = [(n(o, i) * i ** -0.5).to(dtype) for o, i in (((Hq + 2 * Hk) * D, W), (W, Hq * D), (4 * W, W), (W, 4 * W))]
        bs = [n(w.shape[0]) * 0.1 for w in ws]
        off = offsets(lens)
        qkv = ops.linear(x, ws[0], bs[0]).view(T, -1, D)
        att = ops.attention(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], off, causal=True)
        h = ops.linear(att.view(T, Hq * D), ws[1], bs[1], residual=x)
        y = ops.linear(ops.linear(h, ws[2], bs[2], activation="gelu"), ws[3], bs[3], residual=h)
        X, Ws, Bs = x.double(), [w.double() for w in ws], [b.double() for b in bs]
        QKV = (X @ Ws[0].t().contiguous() + Bs[0]).view(T, -1, D)
        A, _ = reference(QKV[:, :Hq], QKV[:, Hq:Hq + Hk], QKV[:, Hq + Hk:], lens, lens, True, D ** -0.5)
        Hh = X + A.reshape(T, -1) @ Ws[1].t().contiguous() + Bs[1]
        z = Hh @ Ws[2].t().contiguous() + Bs[2]
        Y = Hh + (z * torch.special.ndtr(z)) @ Ws[3].t().contiguous() + Bs[3]
        # values of size 1 to 5 through four roundings of 2^-24 / 2^-11 / 2^-8 whose errors add up over sums of 256 and 1024
        # terms: some 30 roundings' worth is the largest a correct chain reaches
        assert float((y.double() - Y).abs().max()) < tol


def test_refusals(vo):
    q, k, v = make([8], [8], 4, 2, 32, torch.float16, 1)
    o = offsets([8])
    bad = [
        (lambda: ops.attention(q.double(), k, v), "float32, float16 or bfloat16"),
        (lambda: ops.attention(q, k.float(), v), "dtype"),
        (lambda: ops.attention(q, k, v.cpu()), "GPU tensor"),
        (lambda: ops.attention(q[0], k, v), "tokens, heads"),
        (lambda: ops.attention(q, k, v[:4]), "k and v"),
        (lambda: ops.attention(q, k[..., :16], v[..., :16]), "k and v"),
        (lambda: ops.attention(q[:, :3], k, v), "multiple"),
        (lambda: ops.attention(q, k, v, None, o), "needs q_offsets"),
        (lambda: ops.attention(q[:4], k, v, o), "as many tokens"),
        (lambda: ops.attention(q, k, v, o.long()), "int32"),
        (lambda: ops.attention(q, k, v, o, offsets([4, 4])), "as many"),
        (lambda: ops.attention(q, k, v, o[:1]), "sequences"),
        (lambda: ops.attention(q, k, v, o.cpu()), "GPU tensor"),
        (lambda: ops.attention(q, k, v, scale=0.0), "scale"),
        (lambda: ops.attention(q, k, v, scale=float("nan")), "scale"),
        (lambda: ops.attention(q, k, v, out=q), "overlaps q"),
        (lambda: ops.attention(q, k, v, out=q[:4]), "out must be"),
        (lambda: ops.attention(q, k, v, out=torch.empty_like(q[:1]).expand(8, 4, 32)), "overlap"),
        (lambda: ops.attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, v), "consecutive"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
    from visual_odometry_amd._lib import VoHipError
    with pytest.raises(VoHipError, match="16-byte pieces"):
        ops.attention(q[..., :20], k[..., :20], v[..., :20])
    with pytest.raises(VoHipError, match="aligned"):
        ops.attention(q[..., 4:28], k[..., 4:28], v[..., 4:28])
    w = torch.zeros(8, 4, 300, device="cuda", dtype=torch.float16)
    with pytest.raises(VoHipError, match="at most 256"):
        ops.attention(w, w, w)


def in_hull(y, v, dtype):
    """Every result is a mean of the values: no further out than their extremes, but for the roundings of the weights (half a step
    each, of 16-bit storage) and of the result, and 2 (n + 64) 2^-24 for the float32 sums of n terms, numerator and denominator."""
    half = torch.finfo(dtype).eps / 2
    slack = 1 + (2 * half + 4 * (len(v) + 64) * U32) * 1.05
    top = v.double().abs().amax(0)
    return bool((y.double().abs() <= top * slack).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("scale", [0.125, 1.0, 1e9, 1e30])
@pytest.mark.parametrize("q_len,k_len", [([140], [300]), ([3], [300]), ([1], [31]), ([140], [4000]), ([3], [4000])])
def test_scores_of_any_size_with_one_key_ahead_give_its_value(vo, dtype, causal, scale, q_len, k_len):
    """Scores up to 4e9, times scales up to 1e30: products of two stored numbers, exact in float32.  The key that is furthest ahead has
    the weight 1, the others' are under e^-100, so the result is its value, bit for bit."""
    lq, lk, D = q_len[0], k_len[0], 64
    q, k, v = make(q_len, k_len, 2, 1, D, dtype, 31)
    q[:], k[:] = 0, 0
    q[..., 7] = 3e4
    g = torch.Generator(device="cuda").manual_seed(8)
    # 256 to 32768 with eight bits each, so that equal ones are equal and different ones 2^-8 of themselves apart (products: 2^13 at least)
    mant = torch.randint(128, 256, (lk,), generator=g, device="cuda").double()
    power = torch.randint(1, 8, (lk,), generator=g, device="cuda").double()
    sign = torch.randint(0, 2, (lk,), generator=g, device="cuda").double() * 2 - 1
    k[:, 0, 7] = (sign * mant * 2 ** power).to(dtype)
    y = ops.attention(q, k, v, causal=causal, scale=scale)
    s = q[0, 0, 7].double() * k[:, 0, 7].double() * scale
    for i in range(lq):
        n = max(0, min(lk, i + 1 + lk - lq)) if causal else lk
        best = s[:n] == s[:n].max()
        others = s[:n][~best]
        assert len(others) == 0 or float(s[:n].max() - others.max()) > 100
        if int(best.sum()) == 1:
            assert torch.equal(y[i], v[int(best.nonzero()[0])].expand(2, D)), i
        else:                                                          # equal keys share the weight
            assert in_hull(y[i], v[:n][best][:, 0], dtype), i


@pytest.mark.parametrize("dtype,spread", [(torch.float32, 6e4), (torch.float32, 1e9), (torch.float16, 1.6e4), (torch.bfloat16, 6e4), (torch.bfloat16, 1e9)])
@pytest.mark.parametrize("q_len,k_len", [([140], [300]), ([3], [300]), ([140], [4000]), ([3], [4000])])
def test_large_random_scores_give_means_of_the_values(vo, dtype, spread, q_len, k_len):
    """Normally distributed queries and keys of a spread near float16's largest numbers, and far over it."""
    g = torch.Generator(device="cuda").manual_seed(9)
    n = lambda *s: (torch.randn(*s, generator=g, device="cuda") * spread).clamp(-6e4 if dtype == torch.float16 else -1e30, 6e4 if dtype == torch.float16 else 1e30)
    q, k = n(q_len[0], 2, 64).to(dtype), n(k_len[0], 1, 64).to(dtype)
    v = (torch.randn(k_len[0], 1, 64, generator=g, device="cuda").abs() + 1).to(dtype)
    y = ops.attention(q, k, v)
    assert in_hull(y, v, dtype) and bool((y.double() >= 0.95).all())        # a row whose weights vanish would give zeros
    # where one key is ahead by more than the scores can be off, its value is the result
    for h in range(2):
        s = q[:, h].double() @ k[:, 0].double().t().contiguous() * 0.125
        b = q[:, h].double().abs() @ k[:, 0].double().abs().t().contiguous() * 0.125
        top = s.topk(2, 1)
        clear = top.values[:, 0] - top.values[:, 1] > 150 + 4 * 66 * U32 * b.amax(1) + 8 * U32 * s.abs().amax(1)
        assert bool(clear.any())
        assert torch.equal(y[clear, h], v[top.indices[clear, 0], 0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("score", ["minus infinity", "underflows"])
@pytest.mark.parametrize("q_len,k_len", [([200], [200]), ([130], [300]), ([140], [2000]), ([5], [90]), ([3], [300]), ([3], [2000])])
def test_an_infinite_value_without_weight_gives_nan_wherever_its_tile_lies(vo, dtype, D, score, q_len, k_len):
    """Zero times infinity, in a tile that every row sees whole, in one on the diagonal and in any part of a split axis: rows that see the
    key have a NaN in that feature and nothing else, the others have nothing of it."""
    lq, lk = q_len[0], k_len[0]
    g = torch.Generator(device="cuda").manual_seed(13)
    for at in sorted({0, 1, lk // 2, max(lk - lq, 0) + lq // 2, lk - 2}):
        q, k, v = make(q_len, k_len, 2, 1, D, dtype, 14 + at)
        q[..., 0] = 4
        k[at, 0] = 0
        k[at, 0, 0] = float("-inf") if score == "minus infinity" else -1000.0        # e^-500 is no float32
        clean = reference(q, torch.cat([k[:at], k[at + 1:]]), torch.cat([v[:at], v[at + 1:]]), [lq], [lk - 1], False, D ** -0.5 if D < 64 else 0.125)
        for causal in (False, True):
            v2 = v.clone()
            v2[at, 0, 3] = float("inf")
            y = ops.attention(q, k, v2, causal=causal, scale=D ** -0.5 if D < 64 else 0.125)
            without = ops.attention(q, k, v, causal=causal, scale=D ** -0.5 if D < 64 else 0.125)
            last = torch.arange(lq, device="cuda") + (lk - lq) if causal else torch.full((lq,), lk - 1, device="cuda")
            sees = last >= at
            alone = (last == 0) & sees                                  # a row's only key: finite scores have the weight 1 there
            want = y[..., 3].isinf() & (alone & (score == "underflows"))[:, None] | y[..., 3].isnan()
            assert bool(want[sees].all()), (at, causal)
            assert torch.equal(y[~sees], without[~sees]), (at, causal)
            y[..., 3] = without[..., 3]                                 # the other features have the same bits, whatever the tile went through
            assert bool(y.isfinite().all()) and torch.equal(y, without), (at, causal)
            if not causal:
                check(without, *clean)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [([140], [140]), ([140], [2000]), ([4], [4]), ([3], [2000])])
def test_rows_whose_only_scores_are_minus_infinity(vo, dtype, q_len, k_len):
    """Zeros under finite values; NaN in the features of values that are not finite."""
    q, k, v = make(q_len, k_len, 1, 1, 32, dtype, 15)
    q[..., 0], k[:] = 4, 0
    k[..., 0] = float("-inf")
    for causal in (False, True):
        assert bool((ops.attention(q, k, v, causal=causal) == 0).all())
    v[0, 0, 3], v[0, 0, 9] = float("inf"), float("nan")
    for causal in (False, True):
        y = ops.attention(q, k, v, causal=causal)
        assert bool(y[..., [3, 9]].isnan().all())
        y[..., [3, 9]] = 0
        assert bool((y == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq", [1, 40, 200])
def test_heads_more_than_16_mib_apart(vo, dtype, lq):
    """A cache with its heads outermost, as a transposed view: 70000 tokens of 128 features lie 17 MiB (float32: 34) apart."""
    n, D = 70000, 128
    g = torch.Generator(device="cuda").manual_seed(17)
    cache = torch.randn(2, 2, n, D, generator=g, device="cuda").to(dtype)
    k, v = cache[0].transpose(0, 1), cache[1].transpose(0, 1)
    assert k.stride(1) * k.element_size() >= 1 << 24
    hold = torch.empty(4, n, D, device="cuda", dtype=dtype)             # queries and results likewise
    hold[:, :lq] = torch.randn(4, lq, D, generator=g, device="cuda").to(dtype)
    q = hold.transpose(0, 1)[:lq]
    out = torch.full((4, n, D), 7.0, device="cuda", dtype=dtype)
    y = ops.attention(q, k, v, causal=True, out=out.transpose(0, 1)[:lq])
    want = ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(y, want) and bool((out[:, lq:] == 7).all())
    check(want[:1], *reference(q[:1], k[:n - lq + 1], v[:n - lq + 1], [1], [n - lq + 1], True, D ** -0.5))


def test_tokens_16_mib_apart_are_refused(vo):
    from visual_odometry_amd._lib import VoHipError
    hold = torch.zeros(3 << 23, device="cuda", dtype=torch.float16)
    far = hold.as_strided((2, 1, 32), (1 << 23, 32, 1))
    near = torch.zeros(2, 1, 32, device="cuda", dtype=torch.float16)
    for args in ((far, near, near), (near, far, near), (near, near, far)):
        with pytest.raises(VoHipError, match="under 16 MiB"):
            ops.attention(*args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[150, 33, 0, 260], [1, 2, 1]])
@pytest.mark.parametrize("order", ["token", "head"])
def test_result_beside_its_inputs_in_one_buffer(vo, dtype, lens, order):
    """The result takes heads of the buffer that holds q, k and v: no element is shared."""
    Hq, Hk, D, T = 4, 2, 64, sum(lens)
    g = torch.Generator(device="cuda").manual_seed(2)
    n = 2 * Hq + 2 * Hk
    hold = torch.randn(T, n, D, generator=g, device="cuda").to(dtype)
    if order == "head":
        hold = hold.transpose(0, 1).contiguous().transpose(0, 1)
    keep = hold.clone()
    q, k, v, out = hold[:, :Hq], hold[:, Hq:Hq + Hk], hold[:, Hq + Hk:Hq + 2 * Hk], hold[:, Hq + 2 * Hk:]
    ops.attention(q, k, v, offsets(lens), causal=True, out=out)
    assert torch.equal(hold[:, :Hq + 2 * Hk], keep[:, :Hq + 2 * Hk])
    check(out, *reference(keep[:, :Hq], keep[:, Hq:Hq + Hk], keep[:, Hq + Hk:Hq + 2 * Hk], lens, lens, True, D ** -0.5))
    for first in (1, Hq - 1, Hq, Hq + Hk, Hq + 2 * Hk - 1):
        with pytest.raises(ValueError, match="overlaps"):
            ops.attention(q, k, v, offsets(lens), causal=True, out=hold[:, first:first + Hq])


@pytest.mark.parametrize("rows,keys,heads", [(1, 3000, 1), (1, 200000, 1), (130, 100000, 1), (1000, 30000, 128), (1, 900, 64)])
def test_float16_keys_far_below_the_first_count_together(vo, rows, keys, heads):
    """One key 18 ahead of all others (e^-18 = 2^-26): one of the others weighs less than float16's smallest number, all of them
    together do not."""
    D = 64
    q = torch.zeros(rows, heads, D, device="cuda", dtype=torch.float16)
    k, v = torch.zeros(keys, 1, D, device="cuda", dtype=torch.float16), torch.zeros(keys, 1, D, device="cuda", dtype=torch.float16)
    q[..., 0], k[0, 0, 0], v[1:] = 1, 18, 1
    y = ops.attention(q, k.expand(keys, heads, D), v.expand(keys, heads, D), scale=1.0).double()
    rest = (keys - 1) * np.exp(-18.0)
    want = rest / (1 + rest)
    # a weight of 2^-26, stored 2^7 up in steps of 2^-24: off by at most half a step, 2^-6 of itself; the float32 sums of n terms; the
    # result's own rounding (2^-25 where it is subnormal)
    assert float((y - want).abs().max()) <= want * (2.0 ** -6 + 2.0 ** -11 + 4 * (keys + 64) * U32) + 2.0 ** -25


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("step", [0, 8, 40])
@pytest.mark.parametrize("q_len,n", [([10], 10), ([3], 10), ([140], 150), ([3], 70)])
def test_tokens_that_overlap_in_memory(vo, dtype, causal, step, q_len, n):
    """Keys and values that are windows of one array; an infinity in it reaches the features in whose place it stands, no others."""
    D, lq = 64, q_len[0]
    q, _, _ = make(q_len, [1], 1, 1, D, dtype, 19)
    g = torch.Generator(device="cuda").manual_seed(20)
    hold = [torch.randn(n * step + 2 * D, generator=g, device="cuda").to(dtype) for _ in range(2)]
    k, v = (h.as_strided((n, 1, D), (step, D, 1)) for h in hold)
    want, tol = reference(q, k, v, q_len, [n], causal, 0.125)
    check(ops.attention(q, k, v, causal=causal), want, tol)
    hold[1][(n - 1) * step + 30] = float("inf")
    y = ops.attention(q, k, v, causal=causal)
    at = torch.isinf(v[:, 0])                                          # (n, D)
    last = torch.arange(lq, device="cuda") + (n - lq) if causal else torch.full((lq,), n - 1, device="cuda")
    hit = (torch.arange(n, device="cuda")[None, :] <= last[:, None]).float() @ at.float() > 0
    assert bool((y[:, 0][hit] == float("inf")).all())
    ok = (y.double() - want).abs()[:, 0] <= tol[:, 0]
    assert bool(ok[~hit].all())


@pytest.mark.parametrize("rows,keys,heads", [(1, 300, 1), (300, 300, 1), (3, 5000, 1), (300, 5000, 1), (1000, 500, 128)])
def test_means_of_float16s_largest_number_stay_finite(vo, rows, keys, heads):
    """One key ahead of many equal ones whose weight, a little over (1 + 2^-11) / 2, rounds up by nearly half a step of float16, while
    the sum that divides them is not rounded: the mean of equal values must not pass them, into infinity where they are the largest."""
    q = torch.zeros(rows, heads, 32, device="cuda", dtype=torch.float16)
    k, v = torch.zeros(keys, 1, 32, device="cuda", dtype=torch.float16), torch.empty(keys, 1, 32, device="cuda", dtype=torch.float16)
    q[..., :2] = 1
    k[1:, 0, 0] = float(np.log(0.5 * (1 + 2.0 ** -11 + 2.0 ** -15)))
    k[1:, 0, 1] = float(np.log(0.5 * (1 + 2.0 ** -11 + 2.0 ** -15))) - float(k[1, 0, 0])
    v[..., :16], v[..., 16:] = 65504, -65504
    y = ops.attention(q, k.expand(keys, heads, 32), v.expand(keys, heads, 32), scale=1.0)
    assert bool(y.isfinite().all())
    assert float((y.double().abs() / 65504 - 1).abs().max()) <= 2.0 ** -10 + 4 * (keys + 64) * U32
    v[0, 0, 5] = float("inf")
    y = ops.attention(q, k.expand(keys, heads, 32), v.expand(keys, heads, 32), scale=1.0)
    assert bool((y[..., 5] == float("inf")).all()) and bool(y[..., 6:].isfinite().all())


def test_between_a_models_features_and_its_correlation(vo):
    """The flow network's own feature rows, attended along their lines of pixels, back into its correlation."""
    from visual_odometry_amd import synthetic as syn
    from visual_odometry_amd.raft.models import RAFTFlow, normalize_image
    from visual_odometry_amd.raft_plugins import gray_batch_to_rgb
    torch.manual_seed(0)
    model = RAFTFlow().cuda().eval()
    left, _ = syn.stereo_sequence(7, 2, 128, 160)
    images = normalize_image(gray_batch_to_rgb(torch.from_numpy(left).cuda()))
    maps = model.features(images)
    B, H, W, C = maps.shape
    rows, heads = maps.reshape(-1, C), 4
    g = torch.Generator(device="cuda").manual_seed(23)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    w1, w2, b1, b2 = n(3 * C, C) * C ** -0.5, n(C, C) * 0.3 * C ** -0.5, n(3 * C) * 0.1, n(C) * 0.1
    qkv = ops.linear(rows, w1, b1).view(-1, 3 * heads, C // heads)
    lines = torch.arange(B * H + 1, device="cuda", dtype=torch.int32) * W
    att = ops.attention(qkv[:, :heads], qkv[:, heads:2 * heads], qkv[:, 2 * heads:], lines, causal=True)
    mixed = ops.linear(att.reshape(-1, C), w2, b2, residual=rows)
    QKV = (rows.double() @ w1.double().t().contiguous() + b1.double()).view(-1, 3 * heads, C // heads)
    A, _ = reference(QKV[:, :heads], QKV[:, heads:2 * heads], QKV[:, 2 * heads:], [W] * (B * H), [W] * (B * H), True, (C // heads) ** -0.5)
    want = rows.double() + A.reshape(-1, C) @ w2.double().t().contiguous() + b2.double()
    # three chained float32 products of 256 terms: 2 (256 + 2) 2^-24 of the magnitudes each, which the weights' exponentials take
    # once more times a score's size; 2^-13 of the largest value is four times that
    assert float((mixed.double() - want).abs().max()) <= 2.0 ** -13 * float(want.abs().max())
    mixed = mixed.view(B, H, W, C)
    low, up = model(images[:1], images[1:], iters=2, fmap1=mixed[:1], fmap2=mixed[1:], normalized=True)
    ref = want.float().view(B, H, W, C)
    low_ref, up_ref = model(images[:1], images[1:], iters=2, fmap1=ref[:1].contiguous(), fmap2=ref[1:].contiguous(), normalized=True)
    assert bool(up.isfinite().all()) and float((up - up_ref).abs().max()) < 0.05
    plain = model(images[:1], images[1:], iters=2, fmap1=maps[:1], fmap2=maps[1:], normalized=True)[1]
    assert float((up - plain).abs().max()) > 0                           # and it is read
