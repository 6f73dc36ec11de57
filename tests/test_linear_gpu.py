"""ops.linear (token-major matrix product with bias, activation and residual in its store) against the definition in
float64, element by element.

Tolerance, derived: the float32 sum of C products is off by at most about C roundings of 2^-24 of the sum of the
products' magnitudes S, in any order (doubled for a matrix instruction whose inner additions round towards zero); every
activation here has a slope of at most 1.13; its own evaluation and the epilogue's additions take a few float32
roundings of the magnitudes involved (16 of them are allowed); the store rounds once, by at most eps / 2 of the value
(and half the smallest subnormal)."""
import math

import pytest
import torch

from visual_odometry_amd import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U32 = 2.0 ** -24


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def check(y, x, w, b=None, act=None, res=None):
    X, W = x.double().reshape(-1, x.shape[-1]), w.double()
    C, K = W.shape[1], W.shape[0]
    z = X @ W.t().contiguous()
    S = X.abs() @ W.abs().t().contiguous()
    bias = torch.zeros(K, device=x.device, dtype=torch.float64) if b is None else b.double()
    z = z + bias
    a = act64(z, act)
    r = torch.zeros_like(a) if res is None else res.double().reshape(-1, K)
    want = a + r
    tiny = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[x.dtype]
    tol = (1.13 * 2 * (C + 2) * U32 * (S + bias.abs()) + 16 * U32 * (z.abs() + a.abs() + r.abs())) * 1.01
    tol = tol + torch.finfo(x.dtype).eps / 2 * (want.abs() + tol) + tiny
    got = y.double().reshape(-1, K)
    assert got.shape == want.shape and y.dtype == x.dtype
    worst = ((got - want).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.3g} times the bound"


def make(M, C, K, dtype, seed, bias=True, res=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return (n(M, C).to(dtype), (n(K, C) * C ** -0.5).to(dtype), n(K) if bias else None, n(M, K).to(dtype) if res else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,C,K", [
    (1, 1, 1), (1, 8, 16), (1, 7, 3), (2, 9, 17), (5, 64, 64), (16, 128, 33), (17, 324, 256), (33, 65, 130), (48, 520, 40), (64, 24, 100),
    (65, 1, 1), (65, 8, 8), (70, 63, 65), (100, 324, 256), (129, 72, 129), (200, 130, 66), (320, 64, 64), (333, 96, 250),
    (1, 4096, 300), (3, 5001, 16), (40, 2056, 24), (70, 4100, 64), (130, 1999, 130),           # split over C
    (1500, 40, 2049), (1543, 33, 2048), (3601, 72, 4001), (3700, 9, 4096),                     # the larger tiles
    (4800, 324, 256),
    (1201, 1003, 1100), (640, 2701, 2700)])                                                    # rows padded to whole pieces first
def test_shapes(vo, dtype, M, C, K):
    x, w, b, r = make(M, C, K, dtype, M * 7 + C * 3 + K, res=True)
    check(ops.linear(x, w), x, w)
    check(ops.linear(x, w, b, "relu", r), x, w, b, "relu", r)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,K", [(3, 40), (90, 72)])
def test_activations_over_their_whole_range(vo, dtype, act, M, K):
    x, w, b, r = make(M, 16, K, dtype, 5, res=True)
    x = (x.float() * torch.logspace(-3, 1.3, M, device="cuda")[:, None]).to(dtype)
    check(ops.linear(x, w, b, act), x, w, b, act)
    check(ops.linear(x, w, None, act, r), x, w, None, act, r)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,C,K", [(9, 72, 40), (96, 72, 40), (1600, 72, 2048), (2, 4096, 24), (1201, 1003, 1100)])
@pytest.mark.parametrize("lead,pad", [(0, 16), (8, 8), (1, 3), (3, 0)])
def test_slices_of_wider_tensors(vo, dtype, M, C, K, lead, pad):
    """x, residual and out are column slices; what lies around out's columns stays as it was."""
    x, w, b, r = make(M, C, K, dtype, 11, res=True)
    wide = lambda t: torch.nn.functional.pad(t, (lead, pad), value=float("nan"))[:, lead:lead + t.shape[1]]
    buf = torch.full((M, lead + K + pad), 7.0, device="cuda", dtype=dtype)
    out = buf[:, lead:lead + K]
    y = ops.linear(wide(x), w, b, "silu", wide(r), out=out)
    assert y is out
    check(out, x, w, b, "silu", r)
    assert bool((buf[:, :lead] == 7).all()) and bool((buf[:, lead + K:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_axes_in_place_residual_and_empty(vo, dtype):
    x, w, b, r = make(2 * 3 * 11, 40, 40, dtype, 3, res=True)
    keep = r.clone()
    y = ops.linear(x.view(2, 3, 11, 40), w, b, "gelu", r.view(2, 3, 11, 40), out=r.view(2, 3, 11, 40))
    assert tuple(y.shape) == (2, 3, 11, 40) and y.data_ptr() == r.data_ptr()
    check(r, x, w, b, "gelu", keep)
    assert tuple(ops.linear(x[:0], w, b).shape) == (0, 40)
    assert tuple(ops.linear(x[0], w, b).shape) == (40,)
    check(ops.linear(x[0], w, b)[None], x[:1], w, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,C,K", [(3, 72, 40), (3, 71, 40), (70, 72, 40), (70, 71, 40), (1500, 72, 2048)])
def test_values_that_are_not_finite_stay_in_their_row(vo, dtype, M, C, K):
    """An infinity or NaN in one row of x (and padding that is NaN behind every row) reaches that row alone."""
    x, w, b, _ = make(M, C, K, dtype, 21)
    hold = torch.full((M + 1, C + 9), float("nan"), device="cuda", dtype=dtype)
    hold[:M, :C] = x
    hold[M // 2, 1] = float("inf")
    hold[M // 2, 2] = float("nan")
    y = ops.linear(hold[:M, :C], w, b)
    assert bool(y[M // 2].isnan().all())
    rest = [i for i in range(M) if i != M // 2]
    check(y[rest], x[rest], w, b)


def test_float16_overflows_to_infinity_and_not_further(vo):
    x = torch.full((2, 64), 200.0, device="cuda", dtype=torch.float16)
    x[1] = 1.0
    w = torch.full((8, 64), 200.0, device="cuda", dtype=torch.float16)
    y = ops.linear(x, w)
    assert bool(y[0].isinf().all()) and bool((y[1] == 12800).all())


@pytest.mark.parametrize("M,C,K", [(1, 4096, 64), (70, 4096, 64), (300, 256, 256)])
def test_equal_inputs_give_equal_bits_also_on_another_stream(vo, M, C, K):
    x, w, b, r = make(M, C, K, torch.bfloat16, 2, res=True)
    want = ops.linear(x, w, b, "gelu", r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [ops.linear(x, w, b, "gelu", r) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(y, want) for y in ys)


@pytest.mark.parametrize("dtype,tiny", [(torch.float32, 2.0 ** -140), (torch.float16, 2.0 ** -24), (torch.bfloat16, 2.0 ** -130)])
@pytest.mark.parametrize("M", [2, 40, 300])
def test_subnormal_values_are_not_flushed(vo, dtype, tiny, M):
    x = torch.zeros(M, 16, device="cuda", dtype=dtype)
    x[:, 3] = tiny * torch.arange(1, M + 1, device="cuda").clamp(max=64)
    w = torch.zeros(24, 16, device="cuda", dtype=dtype)
    w[:, 3] = 1
    assert float(x[0, 3]) > 0 and torch.equal(ops.linear(x, w), x[:, 3:4].expand(M, 24))


@pytest.mark.parametrize("M,C,K", [(3, 8192, 64), (70, 4096, 64), (1201, 1003, 1100)])
def test_two_streams_at_once(vo, M, C, K):
    """Calls that need workspaces, under way on two streams together."""
    sets = [make(M, C, K, torch.float16, 60 + i, res=True) for i in range(2)]
    want = [ops.linear(x, w, b, "gelu", r) for x, w, b, r in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, (st, (x, w, b, r)) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i].append(ops.linear(x, w, b, "gelu", r))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


@pytest.mark.parametrize("M,C,K", [(1, 4096, 64), (70, 4096, 64), (300, 256, 256)])
def test_captured_calls_replay_on_new_contents(vo, M, C, K):
    x, w, b, r = make(M, C, K, torch.float16, 4, res=True)
    ops.linear(x, w, b, "silu", r)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.linear(ops.linear(x, w, b, "silu", r)[:, :K].contiguous(), w[:, :K].contiguous(), b)
    for seed in range(4):
        x2, _, _, r2 = make(M, C, K, torch.float16, 40 + seed, res=True)
        x.copy_(x2); r.copy_(r2)
        g.replay()
        torch.cuda.synchronize()
        want = ops.linear(ops.linear(x, w, b, "silu", r)[:, :K].contiguous(), w[:, :K].contiguous(), b)
        assert torch.equal(y, want)


def test_refusals(vo):
    x, w, b, r = make(8, 16, 24, torch.float16, 1, res=True)
    bad = [
        (lambda: ops.linear(x, w.float()), "dtype"),
        (lambda: ops.linear(x.double(), w.double()), "float32, float16 or bfloat16"),
        (lambda: ops.linear(x[:, :8], w), "rows of 16"),
        (lambda: ops.linear(x, w.t()), "contiguous"),
        (lambda: ops.linear(x, w[:, ::2]), "contiguous"),
        (lambda: ops.linear(x, w, b[:3]), "bias"),
        (lambda: ops.linear(x, w, b.half()), "float32"),
        (lambda: ops.linear(x, w, b, "tanh"), "activation"),
        (lambda: ops.linear(x, w, b, None, r[:4]), "residual"),
        (lambda: ops.linear(x, w, b, None, r.float()), "dtype"),
        (lambda: ops.linear(x, w, out=r[:, :8]), "out must be"),
        (lambda: ops.linear(x.t().contiguous().t(), w), "consecutive"),
        (lambda: ops.linear(x[:1].expand(8, 16), w), "overlap"),
        (lambda: ops.linear(x.view(2, 4, 16).transpose(0, 1), w), "collapse"),
        (lambda: ops.linear(x, w.cpu()), "GPU tensor"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
    buf = torch.zeros(8, 64, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="overlaps x"):
        ops.linear(buf[:, :16], w, out=buf[:, 8:32])
    with pytest.raises(ValueError, match="overlaps residual"):
        ops.linear(x, w, residual=buf[:, :24], out=buf[:, 8:32])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,C,K", [(3, 8, 40), (24, 8, 40), (300, 8, 256), (2, 4096, 40), (70, 4100, 64)])
def test_activations_keep_their_digits_on_the_negative_side(vo, dtype, act, M, C, K):
    """z from -12 (gelu_tanh: -9) to 0, one product of two numbers of eight bits, so exact: the result is right relative to itself, however
    near to zero it is.  An exponential's argument e (z^2 / 2 for gelu, up to 144 / 2) takes at most eight roundings of itself -- gelu:
    |z| / sqrt 2 two, each twice in its square, the square and the change of base one or two each; gelu_tanh: a cube, a sum and
    three factors; silu: two -- and an error of an exponent is a relative one of the result.  2^-20 for the functions themselves and the
    few products around them (16 bits: 2^-19, GELU's polynomial is off by 8e-7); the store's half step, of a subnormal where the result is one."""
    x = torch.zeros(M, C, device="cuda", dtype=dtype)
    w = torch.zeros(K, C, device="cuda", dtype=dtype)
    lo = -12.0 if act != "gelu_tanh" else -9.0
    x[:, 3] = torch.linspace(lo, -0.01, M, device="cuda").bfloat16().to(dtype)                # eight bits each, in every type
    w[:, 3] = (1 - torch.arange(K, device="cuda") / (2.0 * K)).bfloat16().to(dtype)
    z = x[:, 3].double()[:, None] * w[:, 3].double()[None, :]
    if act == "gelu":
        want, e = 0.5 * z * torch.erfc(z * -math.sqrt(0.5)), z * z / 2          # torch's ndtr is (1 + erf) / 2: no digits left at -8
    elif act == "silu":
        want, e = z * torch.sigmoid(z), z.abs()
    else:
        u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        want, e = z * torch.sigmoid(u), u.abs()
    got = ops.linear(x, w, activation=act).double()
    rel = 8 * U32 * (e + 1) + (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -19)
    smallest = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -14, torch.bfloat16: 2.0 ** -126}[dtype]
    half = torch.finfo(dtype).eps / 2
    tol = want.abs() * (rel + half) * 1.01 + smallest * half * 1.01
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1.0, f"error {worst:.3g} times the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M", [3, 40, 300])
def test_activations_of_the_largest_numbers(vo, dtype, act, M):
    """Large numbers and infinity above zero stay as they are, large ones below become zero, NaN stays NaN."""
    big = torch.finfo(dtype).max
    x = torch.tensor([big, float("inf"), -big, float("nan"), 50.0, -300.0], device="cuda").to(dtype).repeat(M // 6 + 1)[:M, None]
    y = ops.linear(x, torch.ones(24, 1, device="cuda", dtype=dtype), activation=act)
    above, below = (x > 0).expand(M, 24), (x < 0).expand(M, 24)
    assert torch.equal(y[above], x.expand(M, 24)[above]) and bool((y[below] == 0).all()) and bool(y[x.isnan().expand(M, 24)].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,C,K", [(1, 40, 24), (9, 72, 40), (96, 71, 33), (1600, 72, 2048), (3, 4096, 64), (1201, 1003, 1100)])
def test_x_residual_and_result_side_by_side_in_one_buffer(vo, dtype, M, C, K):
    """Column ranges of one buffer share no element."""
    x, w, b, r = make(M, C, K, dtype, 13, res=True)
    buf = torch.full((M, C + 2 * K + 3), 7.0, device="cuda", dtype=dtype)
    buf[:, :C], buf[:, C:C + K] = x, r
    ops.linear(buf[:, :C], w, b, "relu", buf[:, C:C + K], out=buf[:, C + K:C + 2 * K])
    check(buf[:, C + K:C + 2 * K], x, w, b, "relu", r)
    assert torch.equal(buf[:, :C], x) and torch.equal(buf[:, C:C + K], r) and bool((buf[:, C + 2 * K:] == 7).all())


def test_columns_that_meet_are_refused(vo):
    """One shared column at either end, across the buffer's line end, or between rows of different strides."""
    x, w, b, r = make(8, 16, 24, torch.float16, 1, res=True)
    buf = torch.zeros(9, 64, device="cuda", dtype=torch.float16)
    flat = buf.view(-1)
    for at in (0, 1, 15, -23, -1):                                      # x in columns 24 .. 39, the result 24 wide at 24 + at
        with pytest.raises(ValueError, match="overlaps x"):
            ops.linear(buf[:8, 24:40], w, out=buf[:8, 24 + at:48 + at])
    ops.linear(buf[:8, 24:40], w, out=buf[:8, 40:64])
    ops.linear(buf[:8, 24:40], w, out=buf[:8, 0:24])
    late = flat[56:56 + 8 * 64].view(8, 64)[:, :16]                     # columns 56 .. 63 and the next row's 0 .. 7
    with pytest.raises(ValueError, match="overlaps x"):
        ops.linear(late, w, out=buf[:8, 0:24])
    with pytest.raises(ValueError, match="overlaps x"):
        ops.linear(late, w, out=buf[:8, 40:64])
    ops.linear(late, w, out=buf[:8, 8:32])
    with pytest.raises(ValueError, match="overlaps x"):
        ops.linear(buf[0:8:2, 0:16], w, out=flat[16:16 + 4 * 40].view(4, 40)[:, :24])
    with pytest.raises(ValueError, match="overlaps weight"):
        ops.linear(x[:2], buf[:6].view(24, 16), out=buf[2:4, :24])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,C,K", [(1, 40, 24), (9, 72, 40), (96, 71, 33), (1600, 72, 2048), (3, 4096, 64), (70, 4100, 64), (1201, 1003, 1100)])
def test_one_residual_row_for_all(vo, dtype, M, C, K):
    """A residual expanded over the rows (their stride is 0)."""
    x, w, b, r = make(M, C, K, dtype, 14, res=True)
    y = ops.linear(x, w, b, "gelu", r[:1].expand(M, K))
    check(y, x, w, b, "gelu", r[:1].expand(M, K))
    assert torch.equal(y, ops.linear(x, w, b, "gelu", r[:1].expand(M, K).contiguous()))
    if M == 96:
        assert torch.equal(ops.linear(x.view(2, 48, C), w, b, "gelu", r[0].expand(2, 48, K)).view(M, K), y)
        with pytest.raises(ValueError, match="out: rows overlap"):
            ops.linear(x, w, out=r[:1].expand(M, K))
        with pytest.raises(ValueError, match="rows overlap"):
            ops.linear(x, w, residual=r.view(-1).as_strided((M, K), (1, 1)))
