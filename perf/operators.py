"""Cases that time the layer operators of the kernel-level C entry points: the
linear layer with bias, activation and residual (inl_cuda_linear), rotary
positions (inl_cuda_rope) and the per-head norms of queries and keys with the
rotation in the same pass (inl_cuda_qk_norm_rotary).

``run`` computes a case with elementary torch operations in 32 bits, or, where
``own`` is true, with the library's kernels. Sizes are those of the towers the
library runs (hidden 768 / 1024, 16 + 8 heads of 128, 12 heads of 64, 3 + 1
heads of 256), their ~64k-token batches and short single queries.
"""
import math

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
DTYPE = {"bf16": BF16, "f32": F32}
# the library's codes
DT = {"f32": 0, "bf16": 1}
ACT = {"silu": 0, "gelu_erf": 1, "gelu_tanh": 2, "none": 3, "relu": 4, "tanh": 5}

MOST_MACS = 65536 * 1024 * 4096  # multiply-adds of the largest listed linear case
MOST_ROWS = 65536 * 24 * 128     # rotated elements of the largest listed rotary cases


# ---------------------------------------------------------------- cases
def _linear(name, M, N, K, dtype, out, act, bias, resid, pad=0):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "out": out, "act": act,
            "bias": bias, "resid": resid, "pad": pad}


def _rope(name, T, heads, d, rot, interleaved, dtype, scaling, theta, far, pad=0):
    return {"name": name, "op": "rope", "T": T, "heads": heads, "d": d, "rot": rot, "interleaved": interleaved,
            "dtype": dtype, "scaling": scaling, "theta": theta, "far": far, "pad": pad}


def _qk(name, T, hq, hkv, d, rot, interleaved, dtype, norm, theta, far):
    return {"name": name, "op": "qk", "T": T, "hq": hq, "hkv": hkv, "d": d, "rot": rot, "interleaved": interleaved,
            "dtype": dtype, "norm": norm, "theta": theta, "far": far}


def listed():
    return [
        # one token's biased q | k | v projection: the smallest call of a serving loop
        _linear("linear_one_token", 1, 4096, 1024, "bf16", "bf16", "none", True, False),
        # a short query's output projection onto the residual stream
        _linear("linear_query_resid", 19, 1024, 2048, "bf16", "bf16", "none", True, True),
        # the MLM head's dense + gelu over a 32-text batch of a 768-wide tower
        _linear("linear_head_gelu", 4253, 768, 768, "bf16", "bf16", "gelu_erf", True, False),
        # a biased, activated projection of an f32 tower over 8 x 128 tokens
        _linear("linear_f32_gelu", 1024, 4096, 1024, "f32", "f32", "gelu_tanh", True, False),
        # sizes no tile divides and rows no vector load aligns with
        _linear("linear_odd", 1531, 1021, 1037, "bf16", "f32", "silu", True, True, 3),
        # the biased q | k | v projection of a 64k-token batch
        _linear("linear_batch", 65536, 4096, 1024, "bf16", "bf16", "none", True, False),
        # one token's query heads
        _rope("rope_one_token", 1, 16, 128, 128, False, "bf16", "yarn", 1e6, 131000),
        # f32 tower, interleaved pairs on half of each 64-wide head, positions scaled for long texts
        _rope("rope_interleaved_part", 20011, 12, 64, 32, True, "f32", "llama3", 5e5, 100000),
        # a 64k-token batch of 16 + 8 heads, rotated by YaRN frequencies
        _rope("rope_batch", 65536, 24, 128, 128, False, "bf16", "yarn", 1e6, 0),
        # a short query through 16 + 8 heads of 128
        _qk("qk_query", 21, 16, 8, 128, 128, False, "bf16", "rms", 1e6, 0),
        # gated-attention heads: 256 wide, a quarter of them rotated, f32
        _qk("qk_part_f32", 4999, 8, 2, 256, 64, False, "f32", "rms", 1e7, 200000),
        # the normed and rotated q / k heads of a 64k-token batch
        _qk("qk_batch", 65536, 16, 8, 128, 128, False, "bf16", "rms", 1e6, 0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above: every size from the smallest calls to the largest batches, odd ones among them."""
    op = rng.choice(["linear", "linear", "rope", "qk"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "linear":
        K, N = _log(rng, 64, 4096), _log(rng, 64, 8192)
        if rng.random() < 0.75:  # what models have; the rest is odd
            K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
        most = MOST_MACS if dtype == "bf16" else MOST_MACS // 8
        M = min(_log(rng, 1, 65536), max(1, most // (N * K)))
        c = _linear("", M, N, K, dtype, dtype if rng.random() < 0.7 else rng.choice(["bf16", "f32"]),
                    rng.choice(list(ACT)), rng.random() < 0.8, rng.random() < 0.4, rng.choice([0, 0, 0, 8, 5]))
    else:
        d = rng.choice([64, 80, 96, 128, 128, 256])
        rot = rng.choice([d, d, d // 2, d // 4])
        inter = rng.random() < 0.4
        hkv = rng.choice([1, 2, 3, 8])
        hq = hkv * rng.choice([1, 2, 4])
        T = min(_log(rng, 1, 65536), max(1, MOST_ROWS // ((hq + hkv) * d)))
        theta, far = rng.choice([1e4, 1.6e5, 5e5, 1e6]), rng.choice([0, 0, 30000, 1000000])
        if op == "rope":
            c = _rope("", T, hq, d, rot, inter, dtype, rng.choice(["none", "linear", "yarn", "llama3"]), theta, far,
                      rng.choice([0, 0, 8, 64, 7]))
        else:
            c = _qk("", T, hq, hkv, d, rot, inter, dtype, rng.choice(["rms", "rms", "layer"]), theta, far)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32)


def _rows(g, rows, cols, pad, dtype, scale=1.0):
    """[rows, cols] values in rows `pad` elements longer than cols."""
    return (_randn(g, rows, cols + pad) * scale).to(dtype)[:, :cols]


def _positions(g, T, far):
    """Positions of packed texts of one to 2048 tokens, the first text's at `far`."""
    lengths = torch.randint(1, 2049, (T // 512 + 2,), generator=g, device="cuda")
    ends = torch.cumsum(lengths, 0)
    t = torch.arange(T, device="cuda")
    text = torch.searchsorted(ends, t, right=True).clamp(max=len(lengths) - 1)
    start = (ends - lengths)[text]
    return (t - start + torch.where(text == 0, far, 0)).to(torch.int32)


def _inv_freq(rot, theta, scaling):
    """Radians per position of each pair, in 64 bits, and the factor on the rotated values."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":  # factor 4 over 32768 positions, 32 and 1 turns
        at = lambda turns: rot * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / 4.0 * ramp, 0.1 * math.log(4.0) + 1.0
    if scaling == "llama3":  # factor 8 over 8192 positions, between 1 and 4 turns
        turns = 8192 * f / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - smooth) * f / 8.0 + smooth * f, 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case, "op": case["op"]}
    dt = DTYPE[case["dtype"]]
    if case["op"] == "linear":
        M, N, K, pad, odt = case["M"], case["N"], case["K"], case["pad"], DTYPE[case["out"]]
        s["x"] = _rows(g, M, K, pad, dt)
        s["w"] = _rows(g, N, K, pad, dt, 1.0 / math.sqrt(K))
        s["bias"] = _randn(g, N) * 0.5 if case["bias"] else None
        s["resid"] = _rows(g, M, N, pad, odt) if case["resid"] else None
        s["out"] = torch.empty(M, N, device="cuda", dtype=odt)
        s["status"] = torch.zeros(1, device="cuda", dtype=torch.int32)
        return s
    T, d = case["T"], case["d"]
    f, scale = _inv_freq(case["rot"], case["theta"], case.get("scaling", "none"))
    s["inv_freq"], s["scale"] = f.cuda(), scale
    s["pos"] = _positions(g, T, case["far"])
    if case["op"] == "rope":
        s["x"] = _rows(g, T, case["heads"] * d, case["pad"], dt)
        s["out"] = torch.empty(T, case["heads"] * d, device="cuda", dtype=dt)
        return s
    hq, hkv = case["hq"], case["hkv"]
    s["qkv"] = _rows(g, T, (hq + 2 * hkv) * d, 0, dt, 2.0)  # packed q | k | v rows, as a projection leaves them
    s["qw"], s["kw"] = 1 + 0.1 * _randn(g, d), 1 + 0.1 * _randn(g, d)
    s["qb"], s["kb"] = (0.1 * _randn(g, d), 0.1 * _randn(g, d)) if case["norm"] == "layer" else (None, None)
    s["q_out"] = torch.empty(T, hq * d, device="cuda", dtype=dt)
    s["k_out"] = torch.empty(T, hkv * d, device="cuda", dtype=dt)
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    return {"linear": _plain_linear, "rope": _plain_rope, "qk": _plain_qk}[s["op"]](s)


def _plain_act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "relu":
        return v.clamp(min=0)
    return torch.tanh(v) if act == "tanh" else v


def _plain_linear(s):
    c = s["case"]
    v = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        v = v + s["bias"]
    v = _plain_act(v, c["act"])
    if s["resid"] is not None:
        v = v + s["resid"].float()
    return v.to(DTYPE[c["out"]])


def _plain_rotate(x, s, c):
    """x [T, heads, d] in 32 bits, its first rot features rotated."""
    rot = c["rot"]
    angle = s["pos"].double()[:, None] * s["inv_freq"]
    cos = (torch.cos(angle) * s["scale"]).float()[:, None]
    sin = (torch.sin(angle) * s["scale"]).float()[:, None]
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    x = s["x"].float().unflatten(-1, (c["heads"], c["d"]))
    return _plain_rotate(x, s, c).flatten(-2).to(s["x"].dtype)


def _plain_head_norm(x, w, b, layer):
    if layer:
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    return y if b is None else y + b


def _plain_qk(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    q = s["qkv"][:, :hq * d].float().unflatten(-1, (hq, d))
    k = s["qkv"][:, hq * d:(hq + hkv) * d].float().unflatten(-1, (hkv, d))
    layer = c["norm"] == "layer"
    q = _plain_rotate(_plain_head_norm(q, s["qw"], s["qb"], layer), s, c)
    k = _plain_rotate(_plain_head_norm(k, s["kw"], s["kb"], layer), s, c)
    return {"q": q.flatten(-2).to(s["qkv"].dtype), "k": k.flatten(-2).to(s["qkv"].dtype)}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    from im_not_llm_b200 import _native
    lib, c = _native.lib(), s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "linear":
        x, w, r, out = s["x"], s["w"], s["resid"], s["out"]
        st = lib.inl_cuda_linear(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), DT[c["dtype"]], c["M"], c["N"],
                                 c["K"], _ptr(s["bias"]), ACT[c["act"]], _ptr(r), 0 if r is None else r.stride(0),
                                 out.data_ptr(), c["N"], DT[c["out"]], s["status"].data_ptr(), stream)
        _native.check(st, "linear")
        return out
    if s["op"] == "rope":
        x, out = s["x"], s["out"]
        st = lib.inl_cuda_rope(x.data_ptr(), x.stride(0), DT[c["dtype"]], c["T"], c["heads"], c["d"], c["rot"],
                               int(c["interleaved"]), s["pos"].data_ptr(), s["inv_freq"].data_ptr(), s["scale"], 0,
                               out.data_ptr(), out.stride(0), stream)
        _native.check(st, "rope")
        return out
    qkv, d, ld = s["qkv"], c["d"], s["qkv"].stride(0)
    q = qkv.data_ptr()
    k = q + c["hq"] * d * qkv.element_size()
    st = lib.inl_cuda_qk_norm_rotary(q, ld, d, k, ld, DT[c["dtype"]], c["T"], c["hq"], c["hkv"], d,
                                     int(c["norm"] == "layer"), s["qw"].data_ptr(), _ptr(s["qb"]), s["kw"].data_ptr(),
                                     _ptr(s["kb"]), 1e-6, c["rot"], int(c["interleaved"]), s["pos"].data_ptr(),
                                     s["inv_freq"].data_ptr(), s["scale"], s["q_out"].data_ptr(), c["hq"] * d,
                                     s["k_out"].data_ptr(), c["hkv"] * d, stream)
    _native.check(st, "qk_norm_rotary")
    return {"q": s["q_out"], "k": s["k_out"]}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = {"bf16": 2, "f32": 4}
    if case["op"] == "linear":
        M, N, K, o = case["M"], case["N"], case["K"], e[case["out"]]
        read = (M * K + N * K) * e[case["dtype"]] + (4 * N if case["bias"] else 0) + (M * N * o if case["resid"] else 0)
        return {"bytes": read + M * N * o, "flops": 2 * M * N * K}
    heads = case["heads"] if case["op"] == "rope" else case["hq"] + case["hkv"]
    n = case["T"] * heads * case["d"]
    flops = 3 * case["T"] * heads * case["rot"] + (0 if case["op"] == "rope" else 4 * n)
    return {"bytes": 2 * n * e[case["dtype"]] + 4 * case["T"] + 4 * case["rot"], "flops": flops}


# ---------------------------------------------------------------- the definition, in 64 bits
def _exact_turn(y, pos, freq, scale, rot, interleaved):
    """Pairs as complex numbers times scale e^(i pos freq)."""
    angle = torch.outer(pos.to(torch.float64), freq)
    turn = torch.polar(torch.full_like(angle, scale), angle).unsqueeze(1)
    pairs = y[..., :rot]
    if interleaved:
        z = torch.view_as_complex(pairs.unflatten(-1, (rot // 2, 2)).contiguous()) * turn
        pairs = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(pairs[..., :rot // 2], pairs[..., rot // 2:]) * turn
        pairs = torch.cat([z.real, z.imag], -1)
    y = y.clone()
    y[..., :rot] = pairs
    return y.flatten(1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = s["x"].to(torch.float64), s["w"].to(torch.float64)
        z = torch.einsum("mk,nk->mn", x, w)
        if s["bias"] is not None:
            z += s["bias"].to(torch.float64)
        act = case["act"]
        if act == "silu":
            z = z * torch.special.expit(z)
        elif act == "gelu_erf":
            z = z * torch.special.ndtr(z)
        elif act == "gelu_tanh":
            z = z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        elif act == "relu":
            z = torch.where(z > 0, z, 0.0)
        elif act == "tanh":
            z = z.tanh_()
        return z if s["resid"] is None else z + s["resid"].to(torch.float64)
    d, turn = case["d"], (s["pos"], s["inv_freq"], s["scale"], case["rot"], case["interleaved"])
    if case["op"] == "rope":
        return _exact_turn(s["x"].to(torch.float64).unflatten(1, (case["heads"], d)), *turn)

    def heads(first, count, w, b):
        y = s["qkv"][:, first * d:(first + count) * d].to(torch.float64).unflatten(1, (count, d))
        if case["norm"] == "layer":
            y = (y - y.mean(-1, keepdim=True)) / torch.sqrt(y.var(-1, unbiased=False, keepdim=True) + 1e-6)
            y = y * w.to(torch.float64) + b.to(torch.float64)
        else:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.to(torch.float64)
        return _exact_turn(y, *turn)

    return {"q": heads(0, case["hq"], s["qw"], s["qb"]), "k": heads(case["hq"], case["hkv"], s["kw"], s["kb"])}
