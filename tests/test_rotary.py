"""inl_cuda_rope, inl_cuda_qk_norm_rotary and inl_cuda_rope_frequencies against
the same formulas in 64 bits, and their refusals.

Tolerances, fixed from the arithmetic, with u = 2^-24 (half a step of f32):
* cos and sin are within 3u of the exact ones (the reduced angle is off by at
  most u, the functions by 1.5u); times the scale, two products and a sum: each
  output is within 8u scale (|a| + |b|) of the rotation of (a, b).
* A normed value is off by (d + 12) u of its size through the mean of d squares
  (d adds, halved by the root) and the products, and for LayerNorm by
  (2 d + 4) u mean|x| / std * |w| through the mean.
* One rounding at the end: u |y| (f32), 2^-8 |y| (bf16).
"""
import ctypes
import math

import numpy as np
import pytest

F32, BF16 = 0, 1
INVALID, CONFIG = 4, 1
U = 2.0 ** -24


def _n():
    from im_not_llm_b200 import _native

    return _native


def _dt(torch, code):
    return torch.bfloat16 if code == BF16 else torch.float32


# ---------------------------------------------------------------- frequencies (CPU)
def _freq(**kw):
    n = _n()
    c = n.RopeConfig(**kw)
    f = np.empty(max(c.rotary_dim // 2, 1))
    scale = ctypes.c_float(-1)
    n.check(n.lib().inl_cuda_rope_frequencies(ctypes.byref(c), f.ctypes.data, ctypes.byref(scale)), "frequencies")
    return f, scale.value


def _base(rot, theta):
    return theta ** (-2.0 * np.arange(rot // 2) / rot)


def test_default_and_linear_frequencies():
    n = _n()
    f, s = _freq(type=n.ROPE_DEFAULT, rotary_dim=128, theta=1e6)
    assert s == 1 and np.allclose(f, _base(128, 1e6), rtol=1e-14)
    f, s = _freq(type=n.ROPE_LINEAR, rotary_dim=64, theta=1e4, factor=8.0)
    assert s == 1 and np.allclose(f, _base(64, 1e4) / 8, rtol=1e-14)
    f, _ = _freq(type=n.ROPE_DEFAULT, rotary_dim=2, theta=1e4)
    assert f.tolist() == [1.0]


def test_dynamic_frequencies():
    n = _n()
    kw = dict(type=n.ROPE_DYNAMIC, rotary_dim=64, theta=1e4, factor=2.0, original_max_position=2048)
    f, s = _freq(seq_len=1000, **kw)  # within the trained length: unscaled
    assert s == 1 and np.allclose(f, _base(64, 1e4), rtol=1e-14)
    f, _ = _freq(seq_len=6144, **kw)
    assert np.allclose(f, _base(64, 1e4 * (2 * 3 - 1) ** (64 / 62)), rtol=1e-13)


def test_yarn_frequencies():
    n = _n()
    rot, theta, orig, factor = 128, 1e6, 32768, 4.0
    f, s = _freq(type=n.ROPE_YARN, rotary_dim=rot, theta=theta, factor=factor, original_max_position=orig)
    b = _base(rot, theta)
    turns = orig * b / (2 * math.pi)  # in the trained length
    assert s == pytest.approx(0.1 * math.log(4) + 1, rel=1e-6)
    fast, slow = turns > 40, turns < 0.8  # beyond the rounded bounds of 32 and 1 turns
    assert fast.sum() > 5 and slow.sum() > 5
    assert np.allclose(f[fast], b[fast], rtol=1e-14) and np.allclose(f[slow], b[slow] / factor, rtol=1e-14)
    low, high = np.floor(rot / 2 * np.log(orig / (32 * 2 * math.pi)) / np.log(theta)), \
        np.ceil(rot / 2 * np.log(orig / (2 * math.pi)) / np.log(theta))
    ramp = np.clip((np.arange(rot // 2) - low) / (high - low), 0, 1)
    assert np.allclose(f, b * (1 - ramp) + b / factor * ramp, rtol=1e-13)
    _, s = _freq(type=n.ROPE_YARN, rotary_dim=rot, theta=theta, factor=40.0, original_max_position=4096, mscale=1.0,
                 mscale_all_dim=0.707)
    assert s == pytest.approx((0.1 * math.log(40) + 1) / (0.0707 * math.log(40) + 1), rel=1e-6)
    _, s = _freq(type=n.ROPE_YARN, rotary_dim=rot, theta=theta, factor=4.0, original_max_position=4096,
                 attention_factor=1.25)
    assert s == 1.25


def test_llama3_frequencies():
    n = _n()
    b = _base(128, 5e5)
    f, s = _freq(type=n.ROPE_LLAMA3, rotary_dim=128, theta=5e5, factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                 original_max_position=8192)
    wave = 2 * math.pi / b
    want = np.where(wave > 8192, b / 8, b)
    mid = (wave <= 8192) & (wave >= 8192 / 4)
    sm = (8192 / wave - 1) / 3
    want = np.where(mid, (1 - sm) * b / 8 + sm * b, want)
    assert s == 1 and mid.any() and np.allclose(f, want, rtol=1e-13)


def test_longrope_frequencies():
    n = _n()
    short, long_ = np.linspace(1, 2, 48), np.linspace(1, 30, 48)
    kw = dict(type=n.ROPE_LONGROPE, rotary_dim=96, theta=1e4, factor=32.0, original_max_position=4096,
              short_factor=short.ctypes.data, long_factor=long_.ctypes.data)
    f, s = _freq(seq_len=4096, **kw)
    assert np.allclose(f, _base(96, 1e4) / short, rtol=1e-14)
    assert s == pytest.approx(math.sqrt(1 + math.log(32) / math.log(4096)), rel=1e-6)
    f, _ = _freq(seq_len=4097, **kw)
    assert np.allclose(f, _base(96, 1e4) / long_, rtol=1e-14)


def test_frequency_refusals():
    n = _n()
    f, s = np.empty(64), ctypes.c_float()

    def code(**kw):
        c = n.RopeConfig(**dict(dict(rotary_dim=64, theta=1e4), **kw))
        return n.lib().inl_cuda_rope_frequencies(ctypes.byref(c), f.ctypes.data, ctypes.byref(s))

    assert code() == 0
    zero = np.zeros(32)
    for bad in (dict(type=6), dict(type=-1), dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=-2),
                dict(theta=0), dict(theta=-1), dict(theta=float("nan")), dict(theta=float("inf")),
                dict(factor=-1, type=1), dict(factor=float("nan"), type=1), dict(type=2), dict(type=3), dict(type=4),
                dict(type=5), dict(type=2, rotary_dim=2, original_max_position=8),
                dict(type=2, factor=0.5, seq_len=100, original_max_position=1, rotary_dim=2),
                dict(type=3, theta=1.0, original_max_position=8),
                dict(type=4, low_freq_factor=4.0, high_freq_factor=4.0, original_max_position=8),
                dict(type=5, original_max_position=8, short_factor=zero.ctypes.data),
                dict(type=5, original_max_position=1, factor=2.0, short_factor=np.ones(32).ctypes.data)):
        assert code(**bad) == INVALID, bad
        assert n.last_error().startswith("rope_frequencies: ")
    assert code(type=5, original_max_position=8) == CONFIG
    assert n.lib().inl_cuda_rope_frequencies(None, f.ctypes.data, ctypes.byref(s)) == CONFIG


# ---------------------------------------------------------------- refusals (CPU)
def test_rope_refusals_need_no_gpu():
    n = _n()

    def call(x=16, ldx=64, dt=BF16, T=2, heads=2, d=32, rot=32, inter=0, pos=16, freq=16, scale=1.0, inv=0, out=32,
             ldo=64):
        return n.lib().inl_cuda_rope(x, ldx, dt, T, heads, d, rot, inter, pos, freq, scale, inv, out, ldo, None)

    for bad in (dict(dt=2), dict(T=-1), dict(T=(1 << 30) + 1), dict(heads=-1), dict(heads=65537, ldx=1 << 30, ldo=1 << 30), dict(d=0), dict(rot=31), dict(rot=34), dict(rot=-2),
                dict(ldx=63), dict(ldo=63), dict(ldx=1 << 41), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(x=17), dict(out=33), dict(pos=18), dict(freq=20), dict(dt=F32, x=18),
                dict(out=16, ldo=128)):
        assert call(**bad) == INVALID, bad
        assert n.last_error().startswith("rope: ")
    for null in (dict(x=None), dict(out=None), dict(pos=None), dict(freq=None)):
        assert call(**null) == CONFIG, null
    assert call(T=0, x=None, out=None, pos=None, freq=None) == 0
    assert call(heads=0, x=None, out=None) == 0


def test_qk_refusals_need_no_gpu():
    n = _n()

    def call(q=16, ldq=96, qhs=32, k=48, ldk=96, dt=BF16, T=2, hq=2, hkv=1, d=32, ln=0, qw=None, qb=None, kw=None,
             kb=None, eps=1e-6, rot=32, inter=0, pos=16, freq=16, scale=1.0, qo=32, ldqo=64, ko=64, ldko=32):
        return n.lib().inl_cuda_qk_norm_rotary(q, ldq, qhs, k, ldk, dt, T, hq, hkv, d, ln, qw, qb, kw, kb, eps, rot,
                                               inter, pos, freq, scale, qo, ldqo, ko, ldko, None)

    for bad in (dict(dt=7), dict(T=-1), dict(hq=-1), dict(hkv=-1), dict(d=0), dict(rot=3), dict(rot=64),
                dict(qhs=31), dict(qhs=128), dict(ldq=63), dict(ldk=31), dict(ldqo=63), dict(ldko=31),
                dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(qb=16), dict(kb=16),
                dict(qw=18), dict(kw=18), dict(k=49), dict(ko=65), dict(ln=1, qb=18),
                dict(qo=16, ldqo=64), dict(qo=16, ldqo=128, ldq=128, qhs=64), dict(ko=48, ldko=32)):
        assert call(**bad) == INVALID, bad
        assert n.last_error().startswith("qk_norm_rotary: ")
    for null in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(pos=None), dict(freq=None)):
        assert call(**null) == CONFIG, null
    assert call(T=0) == 0
    assert call(hq=0, hkv=0, q=None, k=None, qo=None, ko=None) == 0


@pytest.mark.parametrize("d", [(1 << 30) + 1, (1 << 31) - 1])
def test_heads_past_32_bit_feature_indices_are_refused(d):
    n = _n()
    assert n.lib().inl_cuda_rope(16, d, BF16, 1, 1, d, 64, 0, 16, 16, 1.0, 0, 64, d, None) == INVALID
    assert n.last_error() == "rope: T from 0 to 2^30, d from 1 to 2^30"
    assert n.lib().inl_cuda_qk_norm_rotary(16, d, d, 16, d, BF16, 1, 1, 1, d, 0, None, None, None, None, 1e-6, 64, 0, 16, 16, 1.0,
                                           64, d, 64, d, None) == INVALID
    assert n.last_error() == "qk_norm_rotary: T from 0 to 2^30, d from 1 to 2^30"


# ---------------------------------------------------------------- GPU
def _rot64(torch, y, pos, freq, scale, rot, inter, inverse=False):
    """(rotated, sum of the pair's magnitudes) of y [T, heads, d] in 64 bits."""
    ang = pos.double()[:, None] * freq.double()
    c, s = (ang.cos() * scale)[:, None], (ang.sin() * scale * (-1 if inverse else 1))[:, None]
    out, mag = y.clone(), y.abs()
    ia = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
    ib = ia + 1 if inter else ia + rot // 2
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    both = (a.abs() + b.abs()) * abs(scale)
    mag[..., ia], mag[..., ib] = both, both
    return out, mag


def _assert_close(torch, got, want, tol, dt):
    tol = tol + U * want.abs()
    if dt == BF16:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    err = (got.double() - want).abs()
    assert not torch.isnan(got).any()
    assert (err <= tol + 1e-37).all(), (err - tol).max().item()


def _rows(torch, T, width, pad, offset, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((offset + T * (width + pad),), float("nan"), dtype=_dt(torch, dt))
    v = buf[offset:].view(T, width + pad)
    v[:, :width] = torch.randn(T, width, generator=g) * scale
    dev = buf.cuda()
    return dev[offset:].view(T, width + pad)


def _frame(torch, T, width, pad, offset, dt):
    ld = width + pad
    frame = torch.full((offset + (T + 2) * ld,), -55.0, device="cuda", dtype=_dt(torch, dt))
    inside = torch.zeros_like(frame, dtype=torch.bool)
    inside[offset + ld:offset + (T + 1) * ld].view(T, ld)[:, :width] = True
    return frame, frame[offset + ld:offset + (T + 1) * ld].view(T, ld), inside


def _freqs(torch, rot, theta=1e4):
    return torch.tensor(_base(rot, theta), dtype=torch.float64, device="cuda") if rot else None


def _p(t):
    return None if t is None else t.data_ptr()


def _rope(n, torch, x, T, heads, d, rot, inter, pos, freq, scale, inverse, out, dt):
    return n.lib().inl_cuda_rope(x.data_ptr(), x.stride(0), dt, T, heads, d, rot, inter, pos.data_ptr(), _p(freq),
                                 scale, inverse, out.data_ptr(), out.stride(0),
                                 torch.cuda.current_stream().cuda_stream)


ROPES = [  # d, rot, interleaved
    (128, 128, 0), (128, 128, 1), (64, 64, 0), (64, 32, 0), (64, 32, 1), (256, 64, 0), (256, 256, 1), (96, 96, 0),
    (80, 80, 0), (80, 20, 0), (80, 20, 1), (8, 8, 0), (16, 16, 1), (2, 2, 0), (3, 2, 0), (1, 0, 0), (40, 24, 0),
    (576, 64, 1), (300, 150, 0), (128, 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("d,rot,inter", ROPES)
def test_rope(gpu, d, rot, inter, dt):
    import torch

    n = _n()
    for T, heads, pad, offset, opad, scale, inverse in ((1, 1, 0, 0, 0, 1.0, 0), (77, 5, 0, 0, 0, 1.1386, 0),
                                                        (33, 12, 8, 8, 16, 1.0, 1), (70, 3, 3, 1, 5, 0.7, 0)):
        x = _rows(torch, T, heads * d, pad, offset, dt, d + T)
        pos = torch.randint(-5000, 70000, (T,), generator=torch.Generator().manual_seed(T)).int().cuda()
        freq = _freqs(torch, rot)
        frame, out, inside = _frame(torch, T, heads * d, opad, offset, dt)
        before = frame.clone()
        n.check(_rope(n, torch, x, T, heads, d, rot, inter, pos, freq, scale, inverse, out, dt), "rope")
        torch.cuda.synchronize()
        y = x[:, :heads * d].double().unflatten(-1, (heads, d))
        want, mag = y, y.abs()
        if rot:
            want, mag = _rot64(torch, y, pos, freq, scale, rot, inter, inverse)
        _assert_close(torch, out[:, :heads * d].unflatten(-1, (heads, d)), want, 8 * U * mag, dt)
        if rot < d:  # copied features keep their bits
            a, b = out[:, :heads * d].unflatten(-1, (heads, d)), x[:, :heads * d].unflatten(-1, (heads, d))
            assert torch.equal(a[..., rot:], b[..., rot:])
        assert torch.equal(frame[~inside], before[~inside])


# many tokens of few heads (several tokens to a warp), of many (runs of heads), and more than the warps at once
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("T,heads,d,rot,inter", [(2500, 1, 64, 64, 0), (5003, 3, 80, 40, 0), (12001, 4, 64, 32, 1),
                                                 (12001, 1, 128, 128, 0), (5003, 24, 128, 128, 0), (4999, 2, 256, 64, 0),
                                                 (600, 70, 64, 64, 1), (9001, 2, 20, 10, 0), (3001, 1, 8, 8, 0)])
def test_rope_of_many_tokens(gpu, T, heads, d, rot, inter, dt):
    import torch

    n = _n()
    x = _rows(torch, T, heads * d, 8, 0, dt, T)
    pos = torch.randint(0, 100000, (T,), generator=torch.Generator().manual_seed(T)).int().cuda()
    freq = _freqs(torch, rot, 5e5)
    frame, out, inside = _frame(torch, T, heads * d, 8, 0, dt)
    n.check(_rope(n, torch, x, T, heads, d, rot, inter, pos, freq, 1.1, 0, out, dt), "rope")
    torch.cuda.synchronize()
    y = x[:, :heads * d].double().unflatten(-1, (heads, d))
    want, mag = _rot64(torch, y, pos, freq, 1.1, rot, inter)
    _assert_close(torch, out[:, :heads * d].unflatten(-1, (heads, d)), want, 8 * U * mag, dt)
    assert (frame[~inside] == -55).all()
    n.check(_rope(n, torch, x, T, heads, d, rot, inter, pos, freq, 1.1, 0, x, dt), "rope")  # in place
    torch.cuda.synchronize()
    assert torch.equal(x[:, :heads * d], out[:, :heads * d])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("T,hq,hkv,d,rot,inter,ln", [(5003, 2, 1, 64, 64, 0, 0), (12001, 3, 1, 80, 80, 0, 1),
                                                     (9001, 1, 1, 128, 64, 1, 0), (5003, 16, 8, 128, 128, 0, 0),
                                                     (4999, 8, 2, 256, 64, 0, 0), (700, 40, 8, 64, 64, 0, 1)])
def test_qk_of_many_tokens(gpu, T, hq, hkv, d, rot, inter, ln, dt):
    import torch

    n = _n()
    c = dict(hq=hq, hkv=hkv, d=d, rot=rot, inter=inter, ln=ln, eps=1e-6)
    x = _rows(torch, T, (hq + 2 * hkv) * d, 0, 0, dt, d + T, 3.0)
    q, k = x[:, :hq * d], x[:, hq * d:(hq + hkv) * d]
    g = torch.Generator().manual_seed(T)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).cuda() for _ in range(2))
    qb, kb = ((0.2 * torch.randn(d, generator=g)).cuda() for _ in range(2)) if ln else (None, None)
    pos = torch.randint(0, 40000, (T,), generator=g).int().cuda()
    freq = _freqs(torch, rot, 1e6)
    qo, ko = torch.empty(T, hq * d, device="cuda", dtype=x.dtype), torch.empty(T, hkv * d, device="cuda", dtype=x.dtype)
    n.check(_qk(n, torch, c, q, k, d, qw, qb, kw, kb, pos, freq, 1.0, qo, ko, dt, T), "qk")
    torch.cuda.synchronize()
    for src, out, h, w, b in ((q, qo, hq, qw, qb), (k, ko, hkv, kw, kb)):
        v, tol = _norm64(src.double().unflatten(-1, (h, d)), w, b, ln, 1e-6)
        want, mag = _rot64(torch, v, pos, freq, 1.0, rot, inter)
        _assert_close(torch, out.unflatten(-1, (h, d)), want, 8 * U * mag + _rot64(torch, tol, pos, freq, 1.0, rot, inter)[1],
                      dt)


@pytest.mark.gpu
def test_nothing_rotated_reads_no_positions(gpu):
    import torch

    n = _n()
    for d in (64, 7):  # both kernels
        x = _rows(torch, 5, 3 * d, 0, 0, F32, d)
        out = torch.empty_like(x)
        s = torch.cuda.current_stream().cuda_stream
        n.check(n.lib().inl_cuda_rope(x.data_ptr(), 3 * d, F32, 5, 3, d, 0, 0, None, None, 1.0, 0, out.data_ptr(), 3 * d, s),
                "rope")
        torch.cuda.synchronize()
        assert torch.equal(out, x)


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [0, 1])
def test_far_positions_keep_their_digits(gpu, inter):
    import torch

    n = _n()
    T, heads, d = 64, 2, 128
    x = _rows(torch, T, heads * d, 0, 0, F32, 3)
    pos = (torch.arange(T) * 33554393 - 2 ** 30).int()
    pos[0], pos[1] = 2 ** 31 - 1, -2 ** 31
    pos = pos.cuda()
    freq = _freqs(torch, d, 1e6)
    out = torch.empty_like(x)
    n.check(_rope(n, torch, x, T, heads, d, d, inter, pos, freq, 1.0, 0, out, F32), "rope")
    torch.cuda.synchronize()
    want, mag = _rot64(torch, x.double().unflatten(-1, (heads, d)), pos, freq, 1.0, d, inter)
    # 64-bit products of 2^31 are off by up to 2^-22 on either side
    _assert_close(torch, out.unflatten(-1, (heads, d)), want, (8 * U + 2.0 ** -21) * mag, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("d,rot,inter", [(128, 128, 0), (64, 16, 1), (80, 20, 0), (576, 64, 0), (7, 4, 0)])
def test_rope_in_place_and_back(gpu, d, rot, inter, dt):
    import torch

    n = _n()
    T, heads = 41, 6
    x = _rows(torch, T, heads * d, 8, 0, dt, 3)
    pos, freq = torch.arange(T, device="cuda", dtype=torch.int32) * 17, _freqs(torch, rot)
    out = torch.empty(T, heads * d, device="cuda", dtype=_dt(torch, dt))
    orig = x[:, :heads * d].clone()
    n.check(_rope(n, torch, x, T, heads, d, rot, inter, pos, freq, 1.0, 0, out, dt), "rope")
    n.check(_rope(n, torch, x, T, heads, d, rot, inter, pos, freq, 1.0, 0, x, dt), "rope")
    assert torch.equal(x[:, :heads * d], out)  # the same bits in place
    n.check(_rope(n, torch, x, T, heads, d, rot, inter, pos, freq, 1.0, 1, x, dt), "rope")
    torch.cuda.synchronize()
    step = 2.0 ** -8 if dt == BF16 else U
    y = orig.double().unflatten(-1, (heads, d))
    mag = _rot64(torch, y, pos, freq, 1.0, rot, inter)[1]
    err = (x[:, :heads * d].double().unflatten(-1, (heads, d)) - y).abs()
    # two rotations of 8u each and their two roundings, each of at most the pair's magnitude
    assert (err <= (16 * U + 3 * step) * mag * 1.01).all()


def _qk(n, torch, c, q, k, qhs, qw, qb, kw, kb, pos, freq, scale, qo, ko, dt, T):
    s = torch.cuda.current_stream().cuda_stream
    return n.lib().inl_cuda_qk_norm_rotary(_p(q), 0 if q is None else q.stride(0), qhs, _p(k),
                                           0 if k is None else k.stride(0), dt, T, c["hq"], c["hkv"], c["d"], c["ln"],
                                           _p(qw), _p(qb), _p(kw), _p(kb), c["eps"], c["rot"], c["inter"], _p(pos),
                                           _p(freq), scale, _p(qo), 0 if qo is None else qo.stride(0), _p(ko),
                                           0 if ko is None else ko.stride(0), s)


def _norm64(y, w, b, ln, eps):
    """(normed, bound on its error before the rotation) in 64 bits."""
    d = y.shape[-1]
    mean = y.mean(-1, keepdim=True) if ln else 0.0
    z = y - mean
    std = (z.square().mean(-1, keepdim=True) + eps).sqrt()
    wd = 1.0 if w is None else w.double()
    v = z / std * wd
    tol = (d + 12) * U * v.abs()
    if ln:
        tol = tol + (2 * d + 4) * U * y.abs().mean(-1, keepdim=True) / std * (wd.abs() if w is not None else 1.0)
    if b is not None:
        v = v + b.double()
        tol = tol + 2 * U * v.abs()
    return v, tol


QKS = [dict(hq=16, hkv=8, d=128, rot=128, inter=0, ln=0, eps=1e-6), dict(hq=4, hkv=1, d=64, rot=64, inter=1, ln=0, eps=1e-5),
       dict(hq=12, hkv=12, d=64, rot=32, inter=0, ln=1, eps=1e-5), dict(hq=8, hkv=2, d=256, rot=64, inter=0, ln=0, eps=1e-6),
       dict(hq=3, hkv=1, d=256, rot=256, inter=0, ln=1, eps=1e-6), dict(hq=2, hkv=2, d=80, rot=20, inter=0, ln=1, eps=1e-6),
       dict(hq=2, hkv=1, d=96, rot=96, inter=0, ln=0, eps=1e-6), dict(hq=5, hkv=1, d=8, rot=8, inter=0, ln=0, eps=1e-6),
       dict(hq=1, hkv=3, d=13, rot=6, inter=1, ln=1, eps=1e-3), dict(hq=3, hkv=0, d=128, rot=0, inter=0, ln=0, eps=1e-6),
       dict(hq=0, hkv=4, d=32, rot=32, inter=1, ln=0, eps=1e-6), dict(hq=2, hkv=1, d=512, rot=128, inter=0, ln=1, eps=1e-6)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("c", QKS, ids=lambda c: "{hq}-{hkv}-{d}-{rot}-{inter}-{ln}".format(**c))
def test_qk_norm_rotary(gpu, c, dt):
    import torch

    n = _n()
    hq, hkv, d, ln = c["hq"], c["hkv"], c["d"], c["ln"]
    for T, gated, pad, offset, weights in ((1, 0, 0, 0, True), (50, 0, 0, 0, True), (37, 1, 8, 8, True),
                                           (29, 0, 3, 1, True), (13, 0, 0, 0, False)):
        qhs = 2 * d if gated else d
        x = _rows(torch, T, hq * qhs + 2 * hkv * d, pad, offset, dt, d + T, 3.0)
        if ln:
            x += 2.0
        if T > 3:
            x[2, :] = 0.25  # equal features: LayerNorm gives the bias alone
        q = x[:, :hq * qhs] if hq else None
        k = x[:, hq * qhs:(hq * qhs + hkv * d)] if hkv else None
        g = torch.Generator().manual_seed(T)
        vec = lambda m, s: (m + s * torch.randn(d, generator=g)).cuda() if weights else None  # noqa: E731
        qw, kw = vec(1.0, 0.3), vec(1.0, 0.3)
        qb, kb = (vec(0.0, 0.2), vec(0.0, 0.2)) if ln else (None, None)
        pos = torch.randint(0, 40000, (T,), generator=g).int().cuda()
        freq = _freqs(torch, c["rot"], 1e6)
        fq, qo, iq = _frame(torch, T, hq * d, pad, offset, dt)
        fk, ko, ik = _frame(torch, T, hkv * d, pad, offset, dt)
        n.check(_qk(n, torch, c, q, k, qhs, qw, qb, kw, kb, pos, freq, 1.2, qo if hq else None, ko if hkv else None,
                    dt, T), "qk")
        torch.cuda.synchronize()
        for src, out, h, hs, w, b in ((q, qo, hq, qhs, qw, qb), (k, ko, hkv, d, kw, kb)):
            if not h:
                continue
            y = src.double().unflatten(-1, (h, hs))[..., :d]
            v, tol = _norm64(y, w, b, ln, c["eps"])
            want, mag, both = v, v.abs(), tol
            if c["rot"]:
                want, mag = _rot64(torch, v, pos, freq, 1.2, c["rot"], c["inter"])
                both = _rot64(torch, tol, pos, freq, 1.2, c["rot"], c["inter"])[1]
            _assert_close(torch, out[:, :h * d].unflatten(-1, (h, d)), want, 8 * U * mag + both, dt)
        assert (fq[~iq] == -55).all() and (fk[~ik] == -55).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_qk_in_place_captured_and_on_two_streams(gpu, dt):
    import torch

    n = _n()
    c = QKS[0]
    hq, hkv, d, T = c["hq"], c["hkv"], c["d"], 130
    x = _rows(torch, T, (hq + 2 * hkv) * d, 0, 0, dt, 1)
    q, k = x[:, :hq * d], x[:, hq * d:(hq + hkv) * d]
    v0 = x[:, (hq + hkv) * d:].clone()
    w = torch.rand(d, device="cuda") + 0.5
    pos, freq = torch.arange(T, device="cuda", dtype=torch.int32), _freqs(torch, d)
    qo, ko = torch.empty(T, hq * d, device="cuda", dtype=x.dtype), torch.empty(T, hkv * d, device="cuda", dtype=x.dtype)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        n.check(_qk(n, torch, c, q, k, d, w, None, w, None, pos, freq, 1.0, qo, ko, dt, T), "qk")
    graph.replay()
    torch.cuda.synchronize()
    q1, k1 = torch.empty_like(qo), torch.empty_like(ko)
    with torch.cuda.stream(s):
        n.check(_qk(n, torch, c, q, k, d, w, None, w, None, pos, freq, 1.0, q1, k1, dt, T), "qk")
    torch.cuda.synchronize()
    assert torch.equal(q1, qo) and torch.equal(k1, ko)
    n.check(_qk(n, torch, c, q, k, d, w, None, w, None, pos, freq, 1.0, q, k, dt, T), "qk")
    torch.cuda.synchronize()
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(x[:, (hq + hkv) * d:], v0)


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(gpu):
    """A row stride of 2^20 elements over 2100 tokens: the last rows start past 2^31 elements."""
    import torch

    n = _n()
    T, heads, d, ld = 2100, 2, 64, 1 << 20
    buf = torch.zeros(T * ld, device="cuda", dtype=torch.bfloat16)
    x = buf.view(T, ld)[:, :heads * d]
    x.copy_(torch.randn(T, heads * d, generator=torch.Generator().manual_seed(1)))
    pos, freq = torch.arange(T, device="cuda", dtype=torch.int32), _freqs(torch, d)
    out = torch.empty(T, heads * d, device="cuda", dtype=torch.bfloat16)
    want = torch.empty_like(out)
    packed = x.contiguous()
    n.check(_rope(n, torch, x, T, heads, d, d, 0, pos, freq, 1.0, 0, out, BF16), "rope")
    n.check(_rope(n, torch, packed, T, heads, d, d, 0, pos, freq, 1.0, 0, want, BF16), "rope")
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    n.check(_rope(n, torch, packed, T, heads, d, d, 0, pos, freq, 1.0, 0, x, BF16), "rope")
    torch.cuda.synchronize()
    assert torch.equal(x, want)


@pytest.mark.gpu
def test_host_memory_is_refused(gpu):
    import torch

    n = _n()
    d = torch.zeros(2, 8, device="cuda")
    pos, freq = torch.zeros(2, dtype=torch.int32, device="cuda"), _freqs(torch, 8)
    h = torch.zeros(2, 8)
    for x, p, f, o in ((h, pos, freq, d), (d, pos.cpu(), freq, d), (d, pos, freq.cpu(), d), (d, pos, freq, h)):
        assert _rope(n, torch, x, 2, 1, 8, 8, 0, p, f, 1.0, 0, o, F32) == INVALID
        assert "current device" in n.last_error()


@pytest.mark.gpu
def test_projection_norm_rotation_and_attention_together(gpu):
    """One attention block as a caller builds it: the biased q | k | v projection, head norms with a partial YaRN
    rotation in place on the packed rows, attention over packed texts, and the output projection onto the residual
    stream, against the same block in 64 bits. Every bf16 rounding of the block is half a step (2^-9 relative rms at
    most) and the block rounds its values five times; attention averages values and is off by a few steps."""
    import torch

    n = _n()
    N_ = n.lib()
    torch.manual_seed(0)
    H, hq, hkv, d, rot = 256, 4, 2, 64, 32
    lengths = [1, 37, 130, 0, 64]
    cu = np.zeros(len(lengths) + 1, dtype=np.int32)
    np.cumsum(lengths, out=cu[1:])
    T, cols = int(cu[-1]), (hq + 2 * hkv) * d
    h = torch.randn(T, H, device="cuda").bfloat16()
    wqkv = (torch.randn(cols, H, device="cuda") * H ** -0.5).bfloat16()
    bqkv = torch.randn(cols, device="cuda") * 0.5
    wo = (torch.randn(H, hq * d, device="cuda") * (hq * d) ** -0.5).bfloat16()
    bo = torch.randn(H, device="cuda") * 0.5
    qw, kw = torch.rand(d, device="cuda") + 0.5, torch.rand(d, device="cuda") + 0.5
    pos = torch.cat([torch.arange(n_) for n_ in lengths]).int().cuda()
    f, scale = _freq(type=n.ROPE_YARN, rotary_dim=rot, theta=1e4, factor=4.0, original_max_position=64)
    freq = torch.tensor(f, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    qkv = torch.empty(T, cols, device="cuda", dtype=torch.bfloat16)
    n.check(N_.inl_cuda_linear(h.data_ptr(), H, wqkv.data_ptr(), H, BF16, T, cols, H, bqkv.data_ptr(), n.ACT_NONE, None,
                               0, qkv.data_ptr(), cols, BF16, None, s), "qkv")
    c = dict(hq=hq, hkv=hkv, d=d, rot=rot, inter=0, ln=0, eps=1e-6)
    q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
    n.check(_qk(n, torch, c, q, k, d, qw, None, kw, None, pos, freq, scale, q, k, BF16, T), "qk")
    attn = torch.empty(T, hq * d, device="cuda", dtype=torch.bfloat16)
    n.check(N_.inl_cuda_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), cols, cols, cols, attn.data_ptr(), hq * d,
                                  BF16, hq, hkv, d, d ** -0.5, 1, -1, cu.ctypes.data, len(lengths), s), "attention")
    out = h.clone()
    n.check(N_.inl_cuda_linear(attn.data_ptr(), hq * d, wo.data_ptr(), hq * d, BF16, T, H, hq * d, bo.data_ptr(),
                               n.ACT_NONE, out.data_ptr(), H, out.data_ptr(), H, BF16, None, s), "o")
    torch.cuda.synchronize()

    x = h.double() @ wqkv.double().T + bqkv.double()
    q64 = x[:, :hq * d].unflatten(-1, (hq, d))
    k64 = x[:, hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d))
    v64 = x[:, (hq + hkv) * d:].unflatten(-1, (hkv, d))
    q64 = _rot64(torch, _norm64(q64, qw, None, 0, 1e-6)[0], pos, freq, scale, rot, 0)[0]
    k64 = _rot64(torch, _norm64(k64, kw, None, 0, 1e-6)[0], pos, freq, scale, rot, 0)[0]
    o64 = torch.zeros_like(q64)
    for a, b in zip(cu[:-1], cu[1:]):
        if a == b:
            continue
        kk, vv = (t[a:b].repeat_interleave(hq // hkv, 1) for t in (k64, v64))
        sc = torch.einsum("ihd,jhd->hij", q64[a:b], kk) * d ** -0.5
        sc = sc + torch.full_like(sc, float("-inf")).triu(1)
        o64[a:b] = torch.einsum("hij,jhd->ihd", sc.softmax(-1), vv)
    want = h.double() + o64.flatten(1) @ wo.double().T + bo.double()
    rel = ((out.double() - want).norm() / want.norm()).item()
    assert rel < 5 * 2.0 ** -9, rel
