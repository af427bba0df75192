"""inl_cuda_linear (out = act(x w^T + bias) + resid) against the same formula in
64 bits, and its refusals.

Tolerances, fixed from the arithmetic. u = 2^-24 (half a step of f32).
* A sum of K products kept in f32 with each add off by at most a whole step
  (2u of the running value; tensor cores may truncate) is within
  2u (K + 2) S of the exact one, S = sum |x w| + |bias| (element by element).
* The activations' slopes are at most 1.13 (gelu), and they are computed to
  within 2^-19 |v| of the pre-activation value (two hardware approximations of
  2^-22 each, products and sums of a few roundings, with room); a polynomial
  argument or an erf of |v| adds nothing larger.
* One rounding of the result: u |y| (f32) or 2^-9 |y| rounded up to 2^-8 (bf16:
  half a step is 2^-8 of the value below it), plus the residual add's u.
* Norm-wise, independent rounding errors add as sqrt(K): the relative 2-norm
  error of f32 results of random inputs stays below 4 sqrt(K + 16) u.
"""
import ctypes

import pytest

F32, BF16 = 0, 1
ACTS = {"silu": 0, "gelu_erf": 1, "gelu_tanh": 2, "none": 3, "relu": 4, "tanh": 5}
INVALID, CONFIG = 4, 1
U = 2.0 ** -24


def _n():
    from im_not_llm_b200 import _native

    return _native


def _dt(torch, code):
    return torch.bfloat16 if code == BF16 else torch.float32


def _act64(torch, z, act):
    import math

    if act == "silu":
        return z * torch.special.expit(z)
    if act == "gelu_erf":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "relu":
        return torch.relu(z)
    return torch.tanh(z) if act == "tanh" else z


def _rows(torch, rows, cols, pad, dt, seed, scale=1.0, offset=0):
    """rows x cols values inside wider rows whose padding is NaN, `offset` elements into their buffer."""
    g = torch.Generator().manual_seed(seed)
    ld = cols + pad
    buf = torch.full((offset + rows * ld,), float("nan"), dtype=_dt(torch, dt))
    view = buf[offset:].view(rows, ld)[:, :cols]
    view.copy_(torch.randn(rows, cols, generator=g) * scale)
    dev = buf.cuda()
    return dev[offset:].view(rows, ld)[:, :cols], dev


def _call(N, torch, x, w, dt, odt, act, bias, resid, out, stream=None, status=None):
    M, K = x.shape
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    return N.lib().inl_cuda_linear(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), dt, M, w.shape[0], K,
                                   None if bias is None else bias.data_ptr(), ACTS[act],
                                   None if resid is None else resid.data_ptr(),
                                   0 if resid is None else resid.stride(0), out.data_ptr(), out.stride(0), odt,
                                   None if status is None else status.data_ptr(), s)


def _want(torch, x, w, bias, act, resid):
    xd, wd = x.double(), w.double()
    z = xd @ wd.T
    S = xd.abs() @ wd.abs().T
    if bias is not None:
        z, S = z + bias.double(), S + bias.double().abs()
    y = _act64(torch, z, act)
    if resid is not None:
        y = y + resid.double()
    return z, S, y


def _check(torch, got, x, w, bias, act, resid, odt):
    z, S, y = _want(torch, x, w, bias, act, resid)
    K = x.shape[1]
    tol = 1.13 * 2 * U * (K + 2) * S + (0 if act in ("none", "relu") else 2.0 ** -19) * z.abs() + 4 * U * y.abs()
    if resid is not None:
        tol = tol + 2 * U * resid.double().abs()
    if odt == BF16:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs()
    err = (got.double() - y).abs()
    over = (err - tol - 1e-37).max().item() if err.numel() else 0.0
    assert not torch.isnan(got).any()
    assert over <= 0, (over, err.max().item())
    if odt == F32 and y.numel() >= 1024 and act in ("none", "relu", "tanh") and K > 0:
        rel = ((got.double() - y).norm() / y.norm()).item()
        assert rel <= 4 * (K + 16) ** 0.5 * U, rel


def _one(M, N, K, dt, odt, act, bias, resid, pad=(0, 0, 0, 0), offset=0, seed=1):
    import torch

    n = _n()
    x, _ = _rows(torch, M, K, pad[0], dt, seed, 1.0, offset)
    w, _ = _rows(torch, N, K, pad[1], dt, seed + 1, max(K, 1) ** -0.5, offset)
    b = torch.randn(N, generator=torch.Generator().manual_seed(seed + 2)).cuda() if bias else None
    r = _rows(torch, M, N, pad[2], odt, seed + 3, 1.0, offset)[0] if resid else None
    # a frame of a value that the call must leave alone: a row before and after, padding columns, `offset`
    ldo = N + pad[3]
    frame = torch.full((offset + (M + 2) * ldo + 64,), -77.0, device="cuda", dtype=_dt(torch, odt))
    out = frame[offset + ldo:offset + ldo + M * ldo].view(M, ldo)[:, :N]
    before = frame.clone()
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    n.check(_call(n, torch, x, w, dt, odt, act, b, r, out, status=st), "linear")
    torch.cuda.synchronize()
    assert st.item() == 0
    _check(torch, out, x, w, b, act, r, odt)
    inside = torch.zeros_like(frame, dtype=torch.bool)
    inside[offset + ldo:offset + ldo + M * ldo].view(M, ldo)[:, :N] = True
    assert torch.equal(frame[~inside], before[~inside])
    return out


# ---------------------------------------------------------------- CPU
def test_refusals_need_no_gpu():
    n = _n()
    f = n.lib().inl_cuda_linear

    def call(x=16, ldx=8, w=64, ldw=8, dt=BF16, M=2, N=2, K=8, bias=None, act=3, resid=None, ldr=2, out=128, ldo=2,
             odt=BF16, status=None):
        return f(x, ldx, w, ldw, dt, M, N, K, bias, act, resid, ldr, out, ldo, odt, status, None)

    for bad in (dict(dt=2), dict(odt=-1), dict(M=-1), dict(N=-1), dict(K=-1), dict(K=(1 << 30) + 1), dict(act=6),
                dict(act=-1), dict(ldx=7), dict(ldw=7), dict(ldo=1), dict(resid=16, ldr=1), dict(ldx=1 << 41),
                dict(x=17), dict(w=17), dict(out=17), dict(out=16), dict(out=64), dict(bias=18), dict(resid=19), dict(status=2),
                dict(dt=F32, x=18), dict(odt=F32, out=18), dict(resid=128, ldr=4, ldo=2),
                dict(M=1 << 29, N=1 << 29, ldo=1 << 29)):
        assert call(**bad) == INVALID, bad
        assert n.last_error().startswith("linear: ")
    for null in (dict(x=None), dict(w=None), dict(out=None)):
        assert call(**null) == CONFIG, null
        assert "NULL" in n.last_error()
    # nothing to write: no pointer is read
    assert call(M=0, x=None, out=None) == 0
    assert call(N=0, w=None, out=None) == 0


@pytest.mark.parametrize("act", [-1, ACTS["none"], ACTS["relu"], ACTS["tanh"], 6])
def test_gated_products_refuse_the_linear_layers_activations(act):
    """They know silu and the two gelus; another code is not read as one of these."""
    n = _n()
    f = n.lib()
    for epi, block in ((2, 64), (2, 128), (7, 128)):  # INL_GEMM_EPI_GATED, _GATED_F32
        args = n.GemmEx()
        args.A, args.W, args.out, args.lda, args.ldw, args.ldo = 256, 256, 256, 64, 64, 128
        args.M, args.N, args.K, args.epi, args.act, args.gate_block = 8, 256, 64, epi, act, block
        assert f.inl_cuda_gemm_bf16_ex(ctypes.byref(args), None) == INVALID
        assert f.inl_cuda_gemm_bf16(256, 64, 256, 64, 8, 256, 64, epi, act, block, 256, 128, None, 0, 0, None, None) == INVALID
    assert f.inl_cuda_gemm_f32(256, 64, 256, 64, 8, 256, 64, 2, act, 256, 128, None, 0, None) == INVALID


# ---------------------------------------------------------------- GPU
SHAPES = [(1, 1, 1), (1, 4096, 1024), (2, 7, 3), (5, 3, 0), (3, 33, 17), (8, 256, 128), (16, 1000, 520),
          (17, 1024, 2048), (33, 130, 72), (64, 64, 64), (65, 96, 4096), (129, 513, 264), (300, 768, 768),
          (257, 72, 1037), (1000, 1021, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_shapes(gpu, M, N, K, dt):
    _one(M, N, K, dt, dt, "none", True, False)


# sizes on both sides of each choice between the kernels, none of them a multiple of a tile
CHOICES = [  # bf16: few rows, by columns; K shared by clusters of 4 and 2; tiles of 64, 128 and 256 columns, K to 512 and past
    (16, 1180, 136), (9, 2000, 136), (16, 4100, 72), (3, 5000, 264), (32, 1100, 520), (20, 1999, 136), (30, 5001, 136),
    (64, 1150, 328), (100, 1000, 1032), (250, 700, 400), (500, 2300, 320), (500, 2300, 776), (2000, 1000, 200),
    (2000, 1000, 1000), (4200, 760, 520), (4200, 760, 264), (16, 1500, 300), (1900, 1490, 72), (1500, 1500, 1100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,odt,odd", [(BF16, BF16, 0), (BF16, F32, 0), (F32, F32, 0), (F32, BF16, 0), (BF16, BF16, 1),
                                        (F32, F32, 1)])
@pytest.mark.parametrize("M,N,K", CHOICES)
def test_every_choice_of_kernel(gpu, M, N, K, dt, odt, odd):
    _one(M, N, K, dt, odt, "gelu_tanh", True, True, pad=(odd, odd * 3, odd, 5 * odd), seed=21)


# the persistent product's tiles: 64, 128 and 192 columns and the pair's 256, K in one part and in several
TILES = [(500, 2300, 392), (500, 2300, 1096), (2000, 1000, 72), (2000, 1000, 520), (4200, 760, 456), (4200, 760, 776),
         (1281, 577, 1160), (1000, 4090, 1096), (9637, 224, 3832), (500, 2304, 392), (300, 2328, 776),
         (1281, 584, 1160), (1000, 4088, 1096)]


@pytest.mark.gpu
@pytest.mark.parametrize("odt", [BF16, F32])
@pytest.mark.parametrize("act,resid,ragged", [("none", False, 0), ("gelu_erf", True, 0), ("relu", True, 1), ("relu", True, 0),
                                              ("none", True, 8)])
@pytest.mark.parametrize("M,N,K", TILES)
def test_every_tile_of_the_persistent_product(gpu, M, N, K, act, resid, ragged, odt):
    _one(M, N - ragged, K, BF16, odt, act, True, resid, seed=33)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,odt", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [3, 200])
def test_epilogues(gpu, act, dt, odt, M):
    for bias, resid in ((False, False), (True, True), (False, True)):
        _one(M, 320, 192, dt, odt, act, bias, resid, seed=5)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,odt", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("M,N,K", [(4, 96, 200), (150, 264, 200), (260, 520, 136)])
@pytest.mark.parametrize("pad,offset", [((8, 16, 24, 8), 8), ((1, 0, 0, 0), 0), ((0, 3, 0, 0), 0), ((0, 0, 5, 0), 0),
                                        ((0, 0, 0, 7), 0), ((8, 8, 8, 8), 1), ((5, 7, 9, 11), 3)])
def test_strides_and_alignment(gpu, M, N, K, pad, offset, dt, odt):
    _one(M, N, K, dt, odt, "silu", True, True, pad, offset, seed=9)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,odt", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("M,N,K", [(806, 5, 248), (300, 773, 776), (2000, 1003, 72), (4200, 757, 264), (70, 1001, 1032)])
def test_columns_behind_a_row_that_ends_inside_16_bytes_stay(gpu, M, N, K, dt, odt):
    _one(M, N, K, dt, odt, "none", True, False, pad=(8, 8, 0, -N % 8), offset=8)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,odt,M", [(BF16, BF16, 9), (BF16, BF16, 300), (BF16, F32, 300), (F32, F32, 70)])
def test_out_may_be_the_residual(gpu, dt, odt, M):
    import torch

    n = _n()
    N, K = 512, 256
    x, _ = _rows(torch, M, K, 0, dt, 3)
    w, _ = _rows(torch, N, K, 0, dt, 4, K ** -0.5)
    r, _ = _rows(torch, M, N, 8, odt, 5)
    r0 = r.clone()
    n.check(_call(n, torch, x, w, dt, odt, "gelu_erf", None, r, r), "linear")
    torch.cuda.synchronize()
    _check(torch, r, x, w, None, "gelu_erf", r0, odt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("M,N", [(1, 264), (24, 264), (140, 264), (2000, 1500)])
def test_values_that_are_not_finite_stay_in_their_rows(gpu, M, N, dt):
    import torch

    n = _n()
    K = 136
    x, _ = _rows(torch, M, K, 0, dt, 3)
    w, _ = _rows(torch, N, K, 0, dt, 4, 0.1)
    x[0, 5] = float("inf")
    if M > 2:
        x[2, 0] = float("nan")
    out = torch.zeros(M, N, device="cuda", dtype=_dt(torch, dt))
    n.check(_call(n, torch, x, w, dt, dt, "relu", None, None, out), "linear")
    torch.cuda.synchronize()
    want = torch.where(w[:, 5].float() > 0, float("inf"), 0.0)
    assert torch.equal(out[0].float(), want)
    if M > 2:
        assert torch.isnan(out[2]).all()
        rest = [i for i in range(M) if i not in (0, 2)]
        _check(torch, out[rest], x[rest], w, None, "relu", None, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,odt", [(BF16, BF16), (F32, F32)])
def test_captured_on_another_stream_and_replayed(gpu, dt, odt):
    import torch

    n = _n()
    for M in (2, 200):
        N, K = 256, 320
        x, _ = _rows(torch, M, K, 0, dt, 3)
        w, _ = _rows(torch, N, K, 0, dt, 4, K ** -0.5)
        b = torch.randn(N, device="cuda")
        out = torch.empty(M, N, device="cuda", dtype=_dt(torch, odt))
        eager = torch.empty_like(out)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            n.check(_call(n, torch, x, w, dt, odt, "silu", b, None, eager), "linear")
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            st = _call(n, torch, x, w, dt, odt, "silu", b, None, out)
        n.check(st, "linear")
        for seed in (7, 8):
            x.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(seed)))
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            _check(torch, out, x, w, b, "silu", None, odt)
        # two calls in flight on two streams, and the same bits each time
        s2 = torch.cuda.Stream()
        outs = [torch.empty_like(out) for _ in range(4)]
        torch.cuda.synchronize()
        for i, o in enumerate(outs):
            with torch.cuda.stream(s if i % 2 else s2):
                n.check(_call(n, torch, x, w, dt, odt, "silu", b, None, o), "linear")
        torch.cuda.synchronize()
        assert all(torch.equal(o, out) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_rows_past_32_bit_offsets(gpu, dt):
    """Row strides of 2^20 elements over 2100 rows, of x, of the residual and of out: the same bits as of packed rows."""
    import torch

    n = _n()
    M, N, K, ld = 2100, 264, 72, 1 << 20
    x, _ = _rows(torch, M, K, 0, dt, 3)
    w, _ = _rows(torch, N, K, 0, dt, 4, K ** -0.5)
    r, _ = _rows(torch, M, N, 0, dt, 5)
    big = torch.zeros(M * ld, device="cuda", dtype=_dt(torch, dt)).view(M, ld)
    xb, rb, ob = big[:, :K], big[:, 1024:1024 + N], big[:, 2048:2048 + N]
    xb.copy_(x)
    rb.copy_(r)
    out = torch.empty(M, N, device="cuda", dtype=x.dtype)
    n.check(_call(n, torch, x, w, dt, dt, "silu", None, r, out), "linear")
    n.check(_call(n, torch, xb, w, dt, dt, "silu", None, rb, ob), "linear")
    torch.cuda.synchronize()
    assert torch.equal(ob, out) and (big[:, 2048 + N:2048 + N + 64] == 0).all()


@pytest.mark.gpu
def test_memory_the_device_cannot_reach_is_refused(gpu):
    import torch

    n = _n()
    x = torch.zeros(2, 8)
    d = torch.zeros(2, 8, device="cuda")
    o = torch.zeros(2, 2, device="cuda")
    for args in ((x, d[:, :8], o), (d, x, o), (d, d, torch.zeros(2, 2))):
        xx, ww, oo = args
        assert _call(n, torch, xx, ww, F32, F32, "none", None, None, oo) == INVALID
        assert "current device" in n.last_error()
    assert _call(n, torch, d, d, F32, F32, "none", None, None, o) == 0
    pinned = torch.ones(2, 8).pin_memory()  # pinned host memory is reachable
    n.check(_call(n, torch, pinned, torch.ones(2, 8, device="cuda"), F32, F32, "none", None, None, o), "linear")
    torch.cuda.synchronize()
    assert (o == 8).all()


# rows and columns that end inside a warp's 32 x 32 piece of the persistent product's tiles, several pieces to a warp
@pytest.mark.gpu
@pytest.mark.parametrize("odt", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(1937, 1501, 136), (4129, 763, 72), (1503, 2271, 584), (2079, 1025, 648)])
def test_pieces_that_end_inside_a_warp(gpu, M, N, K, odt):
    _one(M, N, K, BF16, odt, "silu", True, True, pad=(-K % 8, -K % 8, 1, 3), seed=41)


# Left of zero gelu and silu fall to 1e-14 of their argument; an f32 result keeps its digits there. The pre-activation
# sum is the bias alone (x is zero), so exact; relative to |y|, by the arithmetic of the formulas in linear.h:
# erfc's argument is off by 2u, times the slope 2 t^2 + 1 = x^2 + 1, its own error 8u (4 ulp), two products: (2 x^2 + 12) u;
# exp's argument w is off by 5u |w|, its own error 4u, a sum and a quotient: (5 |w| + 8) u.
@pytest.mark.gpu
@pytest.mark.parametrize("dt,M,K", [(BF16, 3, 64), (BF16, 130, 1024), (BF16, 700, 64), (BF16, 700, 1024), (F32, 3, 64),
                                    (F32, 130, 1024), (F32, 1500, 64), (BF16, 9, 61), (F32, 150, 61)])
@pytest.mark.parametrize("act", ["silu", "gelu_erf", "gelu_tanh"])
def test_f32_activations_keep_their_digits_on_the_tail(gpu, act, dt, M, K):
    import math

    import torch

    n = _n()
    N = 1500
    x = torch.zeros(M, K, device="cuda", dtype=_dt(torch, dt))
    w = torch.ones(N, K, device="cuda", dtype=_dt(torch, dt))
    v = torch.linspace(-8, 3, N, device="cuda")
    out = torch.empty(M, N, device="cuda")
    n.check(_call(n, torch, x, w, dt, F32, act, v, None, out), "linear")
    torch.cuda.synchronize()
    z = v.double()
    if act == "gelu_erf":
        want, tol = 0.5 * z * torch.special.erfc(-z / math.sqrt(2)), (2 * z * z + 12) * U
    else:
        arg = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        want, tol = z / (1 + torch.exp(-arg)), (5 * arg.abs() + 8) * U
    assert ((out.double() - want).abs() <= tol * want.abs() + 1e-37).all(), ((out.double() - want).abs() / want.abs()).max().item()


# f32 operands that a split into tf32 halves cannot carry: infinities, NaNs and values that round to infinity there, in every
# row and column or in some, through every kernel (few rows; K shared by clusters; tiles walked over; rows of odd strides)
@pytest.mark.gpu
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("M,N,K", [(5, 300, 136), (40, 264, 1100), (140, 264, 520), (1300, 1000, 1100), (2500, 1801, 136)])
@pytest.mark.parametrize("where", ["every row of x", "every row of w", "some of each", "huge"])
def test_f32_values_that_do_not_split(gpu, where, M, N, K, odd):
    import torch

    n = _n()
    inf, nan = float("inf"), float("nan")
    x, _ = _rows(torch, M, K, odd, F32, 3)
    w, _ = _rows(torch, N, K, 3 * odd, F32, 4, 0.01)
    r, _ = _rows(torch, M, N, odd, F32, 5)
    if where == "every row of x":
        x[:, 5] = inf
    elif where == "every row of w":
        w[:, K - 1] = -inf
    elif where == "some of each":
        x[::7, 1], x[3::11, K // 2], x[::7, K - 2], w[::5, 3], w[1, :] = inf, -inf, inf, inf, 0
        x[2, 2], w[4, 2], x[1, 3] = nan, nan, 0
    else:
        x[:, 7], w[::3, 9], x[::2, 9], w[:, 7] = 3.4028e38, -3.4028e38, 1e-3, 0.3
    out = torch.zeros(M, N + odd, device="cuda")[:, :N]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    n.check(_call(n, torch, x, w, F32, F32, "none", None, r, out, status=st), "linear")
    torch.cuda.synchronize()
    z, S, y = _want(torch, x, w, None, "none", r)
    assert st.item() == 0
    # a sum whose products pass f32's range in sum may overflow on the way, or not, by their order: not compared
    sure = ~torch.isfinite(S) | (S <= torch.finfo(torch.float32).max)
    assert torch.equal(torch.isnan(out)[sure], torch.isnan(y)[sure])
    far = torch.isinf(y)
    assert torch.equal(torch.isinf(out)[sure], far[sure]) and torch.equal(out[far].double(), y[far])
    ok = torch.isfinite(y) & sure
    tol = 2 * U * (K + 2) * S[ok] + 4 * U * (y[ok].abs() + r.double()[ok].abs())
    assert ((out.double()[ok] - y[ok]).abs() <= tol + 1e-37).all()


@pytest.mark.gpu
def test_many_long_sums_computed_again_outlast_no_wait(gpu):
    """Every sum of a tile is computed again, for longer than a wait's limit (2 s), while the next tile's products wait for
    its place: that is work, not a wait that ran out."""
    import torch

    n = _n()
    M, N, K = 1024, 4736, 320000
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand(M, K, generator=g, device="cuda")
    w = torch.rand(N, K, generator=g, device="cuda")
    w[::2] *= -1
    x[:, 5] = float("inf")
    out = torch.zeros(M, N, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    n.check(_call(n, torch, x, w, F32, F32, "none", None, None, out, status=st), "linear")
    torch.cuda.synchronize()
    assert st.item() == 0
    assert torch.equal(out, torch.where(w[:, 5] > 0, float("inf"), -float("inf")).expand(M, N))


STALE = """
import ctypes
import numpy as np
import torch
from im_not_llm_b200 import _native as n
lib, one = n.lib(), torch.ones(1, dtype=torch.int32, device="cuda")
x = {0: torch.randn(2000 * 1024, device="cuda")}
x[1] = x[0].bfloat16()
out, f = torch.empty(2000 * 1024, device="cuda"), torch.ones(64, dtype=torch.float64, device="cuda")
pos = torch.zeros(64, dtype=torch.int32, device="cuda")
s = torch.cuda.Stream()
torch.cuda.synchronize()
cu = np.array([0, 4], np.int32)
code = 0
try:  # an allocation inside a capture: the call fails, and so does the capture
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
        code = lib.inl_cuda_causal_conv_silu(x[0].data_ptr(), 8, 8, x[0].data_ptr(), 4, cu.ctypes.data, 1, out.data_ptr(), 8,
                                             s.cuda_stream)
except RuntimeError:
    pass
assert code != 0, "no error was left"
for dt, M, N, K, ld in ((1, 2, 64, 64, 64), (1, 200, 64, 1024, 1024), (1, 2000, 512, 64, 64), (1, 200, 64, 65, 65),
                        (0, 2, 64, 64, 64), (0, 200, 64, 64, 64), (0, 200, 64, 65, 65)):
    code = lib.inl_cuda_linear(x[dt].data_ptr(), ld, x[dt].data_ptr(), ld, dt, M, N, K, None, 3, None, 0, out.data_ptr(), N, 0,
                               None, s.cuda_stream)
    assert code == 0, ("linear", dt, M, N, K, n.last_error())
for dt in (0, 1):
    for ld, off in ((256, 0), (257, 1)):
        p = x[dt].data_ptr() + off * (4, 2)[dt]
        code = lib.inl_cuda_rope(p, ld, dt, 64, 2, 128, 128, 0, pos.data_ptr(), f.data_ptr(), 1.0, 0, out.data_ptr(), 256,
                                 s.cuda_stream)
        assert code == 0, ("rope", dt, ld, n.last_error())
        code = lib.inl_cuda_qk_norm_rotary(p, ld, 128, None, 0, dt, 64, 2, 0, 128, 0, None, None, None, None, 1e-6, 128, 0,
                                           pos.data_ptr(), f.data_ptr(), 1.0, out.data_ptr(), 256, None, 0, s.cuda_stream)
        assert code == 0, ("qk", dt, ld, n.last_error())
torch.cuda.synchronize()
print("fine")
"""


@pytest.mark.gpu
def test_an_earlier_calls_error_is_not_taken_for_a_launchs(gpu):
    """A call of the library that failed leaves its error on the thread; the layer operators after it report their own status.
    In a process of its own, whose capture it spoils."""
    import subprocess
    import sys
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", STALE], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


# Sums of one sign show what an accumulator that truncates loses. A part of c products (512 of K; f32 operands 128) is c / 16
# (f32: c / 8) instructions' worth of truncated adds, each below 2u of a sum that grows evenly: (c / 16 + 1) u of the part;
# the parts are added to nearest, sqrt(K / c) u of the whole in the norm. f32 operands: 2^-21 of each, below 20u, beside.
# Kept in one accumulator the sums are off by 1e-9 K: 74u at 4096, 1100u at 65536 (a warp's share of few rows: 130u).
@pytest.mark.gpu
@pytest.mark.parametrize("K", [4096, 65536])
@pytest.mark.parametrize("dt,odd", [(BF16, 0), (BF16, 1), (F32, 0), (F32, 1)])
@pytest.mark.parametrize("M,N", [(1, 1030), (12, 1100), (14, 5000), (24, 1000), (24, 5000), (50, 1000), (130, 264), (300, 520),
                                 (1000, 264), (520, 2300), (1300, 1000)])
def test_long_sums_of_one_sign(gpu, M, N, dt, odd, K):
    import torch

    n = _n()
    g = torch.Generator(device="cuda").manual_seed(M + N)
    x = (torch.rand(M, K + odd, generator=g, device="cuda") + 0.5).to(_dt(torch, dt))[:, :K]
    w = (torch.rand(N, K + odd, generator=g, device="cuda") + 0.5).to(_dt(torch, dt))[:, :K]
    out = torch.empty(M, N, device="cuda")
    n.check(_call(n, torch, x, w, dt, F32, "none", None, None, out), "linear")
    want = sum(x[:, k:k + 8192].double() @ w[:, k:k + 8192].double().T for k in range(0, K, 8192))
    rel = ((out.double() - want).norm() / want.norm()).item()
    limit = (33 + (K / 512) ** 0.5) * U if dt == BF16 else (17 + 20 + (K / 128) ** 0.5) * U
    assert rel <= limit, (rel / U, limit / U)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1024, 1024), (2048, 640), (1030, 1001)])
def test_long_sums_of_one_sign_in_bf16(gpu, M, N):
    """A bf16 result is the exact sum's rounding but where that lies within the sum's own error e (as above) of a border
    between two: of values spread over their binade, 2 e to a step of 2^-8 of the value at least."""
    import torch

    n = _n()
    K = 1 << 17
    g = torch.Generator(device="cuda").manual_seed(1)
    x = ((torch.rand(M, K, generator=g, device="cuda") + 0.5) * (1 + torch.rand(M, 1, generator=g, device="cuda"))).bfloat16()
    w = (torch.rand(N, K, generator=g, device="cuda") + 0.5).bfloat16()
    for resid in (False, True):
        r = torch.zeros(M, N, device="cuda", dtype=torch.bfloat16) if resid else None
        out, st = torch.empty(M, N, device="cuda", dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32, device="cuda")
        n.check(_call(n, torch, x, w, BF16, BF16, "relu", None, r, out, status=st), "linear")
        want = sum(x[:, k:k + 8192].double() @ w[:, k:k + 8192].double().T for k in range(0, K, 8192))
        assert st.item() == 0
        off = (out != want.bfloat16()).double().mean().item()
        assert off <= 2 * (33 + (K / 512) ** 0.5) * U / 2 ** -8, off
        assert ((out.double() - want).abs() <= 2.0 ** -8 * want).all()


# The residual stream updated in place, through every path that reads the residual ahead of its products or stores: tiles
# of 64 to 256 columns, K in one part and in several, clusters, few rows, rows of odd strides, ragged last tiles.
@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu_tanh"])
@pytest.mark.parametrize("dt,odt,odd", [(BF16, BF16, 0), (BF16, F32, 0), (BF16, BF16, 1), (BF16, F32, 1), (F32, F32, 0),
                                        (F32, BF16, 0), (F32, F32, 1)])
@pytest.mark.parametrize("M,N,K", [(1, 520, 136), (16, 1176, 136), (30, 5000, 136), (64, 1152, 328), (100, 1000, 1032),
                                   (250, 704, 400), (500, 2304, 392), (500, 2304, 776), (2001, 1000, 200),
                                   (2001, 1000, 1000), (4205, 760, 264), (4205, 760, 520), (1283, 584, 1160),
                                   (1003, 4088, 1096), (515, 515, 72), (70, 264, 33000)])
def test_the_residual_updated_in_place(gpu, M, N, K, dt, odt, odd, act):
    import torch

    n = _n()
    x, _ = _rows(torch, M, K, odd, dt, 3)
    w, _ = _rows(torch, N, K, odd, dt, 4, K ** -0.5)
    b = torch.randn(N, generator=torch.Generator().manual_seed(6)).cuda()
    r, frame = _rows(torch, M, N, 16 + odd, odt, 5)
    r0, st = r.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
    n.check(_call(n, torch, x, w, dt, odt, act, b, r, r, status=st), "linear")
    torch.cuda.synchronize()
    assert st.item() == 0 and torch.isnan(frame.view(M, -1)[:, N:]).all()
    _check(torch, r, x, w, b, act, r0, odt)


# A bf16 result's gelu (erf): 2^-19 of the value (the fit, the exponential's argument at most (x^2 + 1) 2^-23 = 2^-17 at -8)
# before one rounding, where the sum is exact (x is zero, the bias is it). Values from -8 up, so the tail counts.
@pytest.mark.gpu
@pytest.mark.parametrize("dt,M,K", [(BF16, 3, 64), (BF16, 130, 1024), (BF16, 700, 64), (F32, 3, 64), (F32, 1500, 64),
                                    (BF16, 150, 61)])
def test_bf16_gelu_keeps_its_digits_on_the_tail(gpu, dt, M, K):
    import math

    import torch

    n = _n()
    N = 1504
    x = torch.zeros(M, K, device="cuda", dtype=_dt(torch, dt))
    w = torch.ones(N, K, device="cuda", dtype=_dt(torch, dt))
    v = torch.linspace(-8, 3, N, device="cuda")
    out = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
    n.check(_call(n, torch, x, w, dt, BF16, "gelu_erf", v, None, out), "linear")
    torch.cuda.synchronize()
    z = v.double()
    want = 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    before = (2.0 ** -19 + (z * z + 1) * 2.0 ** -23) * want.abs()
    assert ((out.double() - want).abs() <= before * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 1e-37).all()


# bf16 results of long K, whose sums come in parts: tiles of 64, 128, 192 and the pair's 256 columns, rows of any alignment
@pytest.mark.gpu
@pytest.mark.parametrize("M,N,resid,pad", [(1024, 1024, True, 0), (1500, 1500, True, 0), (2040, 1728, False, 8),
                                           (2048, 2040, True, 0), (2000, 1999, True, 3)])
def test_bf16_results_of_long_k(gpu, M, N, resid, pad):
    _one(M, N, 32776, BF16, BF16, "gelu_erf", True, resid, pad=(0, 0, pad, pad), seed=51)
