"""The steps of a DSA attention layer on either side of its cache and query, as cases that can be timed and checked:
the RMS norm that hands 8-bit activations to a projection, the projection on FP8 block-scaled weights, the rotary
positions of the query, and the cache row of a token's latent (norm, rotary, quantization and write).

    own                  whether run() calls this package's operators or their plain forms in torch
    listed()             the cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  the inputs, weights, frequencies and caches that a serving program holds before the call
    run(state)           one call and its outputs
    work(case)           bytes and operations that the call cannot do without
    exact(case, seed)    the outputs in 64 bits
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
LAT, ROPE = 512, 64                # latent and rotary widths of a cache row
GROUP = 128                        # values per activation scale, and the side of a weight's scale block
E4M3_MAX = 448.0
S_MIN = 1e-12                      # smallest activation scale (rows of zeros)
KV_SCALE = 0.25                    # per-tensor scale of the fp8 (576-byte) cache
QKV_A = 2112                       # columns of the joint down projection: 1536 of the query, 512 + 64 of the cache
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one user's token enters a layer: residual added, norm, 8-bit activations for the down projection
        dict(name="norm_1", kind="norm", tokens=1, dim=4096, stride=4096, residual=True, fp8=True, ue8m0=False,
             dtype="bf16"),
        # a decode batch's query latents, a slice of the joint down projection's rows
        dict(name="norm_64_slice", kind="norm", tokens=64, dim=1536, stride=QKV_A, residual=False, fp8=True,
             ue8m0=False, dtype="bf16"),
        # a prefill chunk enters a layer, scales rounded up to powers of two
        dict(name="norm_prefill", kind="norm", tokens=8192, dim=4096, stride=4096, residual=True, fp8=True, ue8m0=True,
             dtype="bf16"),
        # one user's token through the joint down projection
        dict(name="linear_1", kind="linear", tokens=1, cols=QKV_A, k=4096, quant=False, dtype="bf16"),
        # a decode batch through the query's up projection (128 heads of 128 + 64)
        dict(name="linear_64", kind="linear", tokens=64, cols=24576, k=1536, quant=False, dtype="bf16"),
        # a decode batch through the attention's output projection, from bf16 (quantized in the call)
        dict(name="linear_out_32", kind="linear", tokens=32, cols=4096, k=16384, quant=True, dtype="bf16"),
        # a ragged chunk of several prompts through the down projection
        dict(name="linear_ragged", kind="linear", tokens=1455, cols=QKV_A, k=4096, quant=False, dtype="bf16"),
        # a prefill chunk through the output projection
        dict(name="linear_prefill", kind="linear", tokens=4096, cols=4096, k=16384, quant=False, dtype="bf16"),
        # a decode batch's rotary query part into the attention's query buffer, positions scaled for long contexts
        dict(name="rope_64", kind="rope", tokens=64, heads=128, width=64, rot=64, start=0, pitch=192, out_pitch=576,
             interleaved=True, scaled=True, dtype="bf16"),
        # a prefill chunk's indexer queries: the first half of each head turns, half layout
        dict(name="rope_prefill", kind="rope", tokens=8192, heads=64, width=128, rot=64, start=0, pitch=128,
             out_pitch=128, interleaved=False, scaled=False, dtype="bf16"),
        # a padded decode batch's cache rows
        dict(name="latent_64", kind="latent", tokens=64, rows=65536, row=656, padded=8, interleaved=True, scaled=True),
        # a prefill chunk's cache rows, per-tensor fp8 cache
        dict(name="latent_prefill", kind="latent", tokens=8192, rows=65536, row=576, padded=0, interleaved=True,
             scaled=False),
    ]


def _logu(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "linear", "linear", "linear", "rope", "rope", "latent"])
    if kind == "norm":
        dim = _logu(rng, 128, 8192)
        dim = dim if rng.random() < 0.3 else dim // 8 * 8
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = _logu(rng, 1, min(8192, (1 << 25) // dim))
        return dict(kind="norm", tokens=tokens, dim=dim, stride=dim + rng.choice([0, 0, 64, 576]),
                    residual=rng.random() < 0.6, fp8=rng.random() < 0.7, ue8m0=rng.random() < 0.3, dtype=dtype)
    if kind == "linear":
        cols, k = _logu(rng, 64, 24576), _logu(rng, 32, 1024) * 16
        tokens = _logu(rng, 1, min(4096, (1 << 38) // (cols * k)))
        return dict(kind="linear", tokens=tokens, cols=cols, k=k, quant=rng.random() < 0.3,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "rope":
        width = rng.choice([64, 128, 192, 256, 80])
        rot = width if width == 64 else rng.choice([width, 64, width // 2])
        heads = rng.choice([1, 5, 8, 32, 64, 128])
        pitch = width + rng.choice([0, 0, 64, 128])
        return dict(kind="rope", tokens=_logu(rng, 1, min(8192, (1 << 26) // (heads * width))), heads=heads,
                    width=width, rot=rot, start=rng.choice([0, width - rot]), pitch=pitch,
                    out_pitch=rng.choice([width, pitch]), interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    tokens = _logu(rng, 1, 8192)
    return dict(kind="latent", tokens=tokens, rows=rng.randrange(8192, 65536), row=rng.choice([656, 576]),
                padded=rng.choice([0, 0, tokens // 8]), interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------- inputs from the seed
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV, dtype=torch.float32)


def _activations(g, tokens, dim):
    """Hidden states: each token at its own size, a few channels far above the others."""
    x = _randn(g, tokens, dim) * torch.exp(0.5 * _randn(g, tokens, 1))
    return x * torch.where(_rand(g, dim) < 0.004, 20.0, 1.0)


def _norm_weight(g, dim):
    return 1.0 + 0.2 * _randn(g, dim)


def _frequencies(rot, scaled):
    """Radians a position, float64 [rot / 2], and the factor of cos and sin. scaled: a context of 4096 positions
    stretched 40 times, low frequencies divided by 40, high ones kept, a ramp between those that turn 32 times and
    once within 4096 positions."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    f = 10000.0 ** (-2.0 * i / rot)
    if not scaled:
        return f, 1.0
    at = lambda turns: rot * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(10000.0))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return f / 40.0 * ramp + f * (1.0 - ramp), 0.1 * math.log(40.0) + 1.0


def _positions(g, tokens, scaled):
    """Decode: a position of its own for each token; a chunk: consecutive ones. Long contexts where scaled."""
    far = 163840 if scaled else 65536
    if tokens <= 256:
        return torch.randint(0, far, (tokens,), generator=g, device=DEV)
    at = torch.randint(0, far - tokens, (1,), generator=g, device=DEV)
    return at + torch.arange(tokens, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, T = case["kind"], case["tokens"]
    s = dict(case=case)
    if kind == "norm":
        dt, D = TYPES[case["dtype"]], case["dim"]
        s["x"] = torch.nn.functional.pad(_activations(g, T, D), (0, case["stride"] - D)).to(dt)[:, :D]
        s["weight"] = _norm_weight(g, D).to(dt)
        s["residual"] = _activations(g, T, D).to(dt) if case["residual"] else None
        s["residual_out"] = torch.empty(T, D, dtype=dt, device=DEV) if case["residual"] else None
        if case["fp8"]:
            s["codes"] = torch.empty(T, D, dtype=torch.float8_e4m3fn, device=DEV)
            s["scales"] = torch.empty(T, -(-D // GROUP), dtype=torch.float32, device=DEV)
        else:
            s["out"] = torch.empty(T, D, dtype=dt, device=DEV)
    elif kind == "linear":
        N, K, dt = case["cols"], case["k"], TYPES[case["dtype"]]
        nb, kb = -(-N // GROUP), -(-K // GROUP)
        s["w"] = (105.0 * _randn(g, N, K)).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        s["w_scales"] = 2e-4 * torch.exp(0.3 * _randn(g, nb, kb))
        x = _activations(g, T, K).to(dt)
        if case["quant"]:
            s["x"] = x
        else:
            s["a"], s["a_scales"] = _quantized(x.float(), False)
        s["out"] = torch.empty(T, N, dtype=dt, device=DEV)
    elif kind == "rope":
        H, W, dt = case["heads"], case["width"], TYPES[case["dtype"]]
        s["x"] = _randn(g, T, H, case["pitch"]).to(dt)[..., case["pitch"] - W:]
        s["out"] = torch.zeros(T, H, case["out_pitch"], dtype=dt, device=DEV)[..., case["out_pitch"] - W:]
        s["positions"] = _positions(g, T, case["scaled"])
        s["freqs"], s["factor"] = _frequencies(case["rot"], case["scaled"])
    else:
        R, row = case["rows"], case["row"]
        s["kv"] = _activations(g, T, QKV_A).to(torch.bfloat16)[:, QKV_A - LAT - ROPE:]
        s["weight"] = _norm_weight(g, LAT).to(torch.bfloat16)
        s["positions"] = _positions(g, T, case["scaled"])
        s["freqs"], s["factor"] = _frequencies(ROPE, case["scaled"])
        s["slots"] = _slots(case, g)
        s["pool"] = torch.zeros(R + 1, row, dtype=torch.uint8, device=DEV)       # the row behind the cache: scratch
        s["pool"][:, :LAT] = torch.randint(0, 120, (R + 1, 1), generator=g, device=DEV).to(torch.uint8)
        s["cache"] = s["pool"][:R]
    return s


def _slots(case, g):
    """Distinct rows in no order; the padded tokens at the end have none (-1)."""
    slots = torch.randperm(case["rows"], generator=g, device=DEV)[:case["tokens"]]
    slots[case["tokens"] - case["padded"]:] = -1
    return slots


# ---------------------------------------------------------------------------------------------- one call
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from arcagi2_flashnext_dots3_amd import kernels, mla_fp8
    c = s["case"]
    if c["kind"] == "norm":
        if c["fp8"]:
            kernels.rms_norm_fp8(s["x"], s["weight"], EPS, residual=s["residual"], residual_out=s["residual_out"],
                                 codes=s["codes"], scales=s["scales"], ue8m0=c["ue8m0"])
            return _given(s, "codes", "scales", "residual_out")
        kernels.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], residual_out=s["residual_out"],
                         out=s["out"])
        return _given(s, "out", "residual_out")
    if c["kind"] == "linear":
        x = s["x"] if c["quant"] else (s["a"], s["a_scales"])
        return mla_fp8.linear_fp8(x, (s["w"], s["w_scales"]), out=s["out"])
    if c["kind"] == "rope":
        return kernels.rope(s["x"], s["positions"], s["freqs"], out=s["out"], start=c["start"],
                            interleaved=c["interleaved"], factor=s["factor"])
    kernels.latent_write(s["kv"], s["weight"], EPS, s["positions"], s["freqs"], s["slots"], s["cache"],
                         fmt=0 if c["row"] == 656 else 1, kv_scale=KV_SCALE, interleaved=c["interleaved"],
                         factor=s["factor"])
    return _rows(s["cache"])


def _given(s, *names):
    return {n: s[n] for n in names if s.get(n) is not None}


def _rows(cache):
    """The cache's values: e4m3 codes, group scales and rotary parts, as views of its rows."""
    if cache.shape[1] == 576:
        return {"codes": cache.view(torch.float8_e4m3fn)}
    return {"codes": cache[:, :LAT].view(torch.float8_e4m3fn), "scales": cache[:, LAT:LAT + 16].view(torch.float32),
            "rope": cache[:, LAT + 16:].view(torch.bfloat16)}


def _quantized(y, ue8m0):
    """y [T, D] fp32 -> e4m3 codes [T, D] and fp32 scales, one per 128 values: largest magnitude / 448."""
    T, D = y.shape
    G = -(-D // GROUP)
    groups = torch.nn.functional.pad(y, (0, G * GROUP - D)).view(T, G, GROUP)
    sc = (groups.abs().amax(2).double() / E4M3_MAX).clamp_min(S_MIN)   # (64 bits: many quotients lie halfway between
    if ue8m0:                                                          # two codes)
        m, e = torch.frexp(sc)                                    # sc = m 2^e, 0.5 <= m < 1
        sc = torch.ldexp(torch.ones_like(sc), torch.where(m > 0.5, e, e - 1))
    codes = (groups.double() / sc[:, :, None]).float().to(torch.float8_e4m3fn)
    return codes.view(T, G * GROUP)[:, :D].contiguous(), sc.float()


def _normed(z, weight):
    return z * torch.rsqrt(z.square().mean(1, keepdim=True) + EPS) * weight.float()


def _turned(x, positions, freqs, factor, start, interleaved):
    """x [T, H, W] fp32 with the pairs of columns start .. start + 2 len(freqs) turned by position * frequency."""
    n = freqs.shape[0]
    angle = positions.double()[:, None] * freqs
    cos, sin = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    part = x[..., start:start + 2 * n]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), 3).flatten(2) if interleaved else torch.cat((u, v), 2)
    return torch.cat((x[..., :start], turned, x[..., start + 2 * n:]), 2)


def _plain(s):
    c = s["case"]
    if c["kind"] == "norm":
        z, got = s["x"].float(), {}
        if c["residual"]:
            s["residual_out"].copy_(z + s["residual"].float())
            z = s["residual_out"].float()
            got["residual_out"] = s["residual_out"]
        y = _normed(z, s["weight"])
        if c["fp8"]:
            got["codes"], got["scales"] = _quantized(y, c["ue8m0"])
        else:
            got["out"] = y.to(s["x"].dtype)
        return got
    if c["kind"] == "linear":
        a, sa = _quantized(s["x"].float(), False) if c["quant"] else (s["a"], s["a_scales"])
        N, K = s["w"].shape
        af = a.float() * sa.repeat_interleave(GROUP, 1)[:, :K]
        ws = s["w_scales"].repeat_interleave(GROUP, 0)[:N].repeat_interleave(GROUP, 1)[:, :K]
        return (af @ (s["w"].float() * ws).t()).to(s["out"].dtype)
    if c["kind"] == "rope":
        y = _turned(s["x"].float(), s["positions"], s["freqs"], s["factor"], c["start"], c["interleaved"])
        s["out"].copy_(y)
        return s["out"]
    lat = _normed(s["kv"][:, :LAT].float(), s["weight"])
    pe = _turned(s["kv"][:, None, LAT:].float(), s["positions"], s["freqs"], s["factor"], 0, c["interleaved"])[:, 0]
    if c["row"] == 656:
        codes, sc = _quantized(lat, False)
        rows = torch.cat((codes.view(torch.uint8), sc.view(torch.uint8), pe.to(torch.bfloat16).view(torch.uint8)), 1)
    else:
        v = torch.cat((lat, pe), 1) / KV_SCALE
        rows = v.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    s["pool"][torch.where(s["slots"] < 0, c["rows"], s["slots"])] = rows
    return _rows(s["cache"])


# ---------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    T, kind = case["tokens"], case["kind"]
    if kind == "norm":
        D, e = case["dim"], TYPES[case["dtype"]].itemsize
        moved = T * D * e * (3 if case["residual"] else 1) + D * e
        moved += T * D + 4 * T * -(-D // GROUP) if case["fp8"] else T * D * e
        return {"bytes": moved, "flops": 4 * T * D}
    if kind == "linear":
        N, K, e = case["cols"], case["k"], 2
        a = T * K * e if case["quant"] else T * K + 4 * T * -(-K // GROUP)
        return {"bytes": a + N * K + 4 * -(-N // GROUP) * -(-K // GROUP) + T * N * e, "flops": 2 * T * N * K}
    if kind == "rope":
        n = T * case["heads"] * case["width"]
        return {"bytes": 2 * n * TYPES[case["dtype"]].itemsize + 8 * T + 4 * case["rot"],
                "flops": 3 * T * case["heads"] * case["rot"]}
    n = T - case["padded"]
    return {"bytes": n * (2 * (LAT + ROPE) + 8 + case["row"]) + 8 * T + 2 * LAT, "flops": n * (4 * LAT + 3 * ROPE)}


# ---------------------------------------------------------------------------------------------- the outputs in 64 bits
def _code_values(q):
    """The e4m3 values of q (float64), to nearest, ties to even: 3 bits of mantissa, steps of 2^-9 at least."""
    _, e = torch.frexp(q)
    step = torch.ldexp(torch.ones_like(q), (e - 4).clamp(min=-9))
    return torch.round(q / step) * step


def _groups64(t, r, ue8m0):
    """Code values and scales of y = t r (t float64 [T, D], r one factor a token). A group's largest magnitude becomes
    448 whatever r is, so the quotients are taken without it: those halfway between two codes stay exactly there."""
    codes, scales = [], []
    for i in range(0, t.shape[1], GROUP):
        p = t[:, i:i + GROUP]
        top = p.abs().max(dim=1, keepdim=True).values
        sc = top * r / E4M3_MAX
        low = sc < S_MIN
        sc = torch.where(low, S_MIN, sc)
        q = torch.where(low, p * r / S_MIN, p * E4M3_MAX / torch.where(low, 1.0, top))
        if ue8m0:
            sc = torch.exp2(torch.ceil(torch.log2(sc)))
            q = p * r / sc
        codes.append(_code_values(q))
        scales.append(sc)
    return torch.cat(codes, 1), torch.cat(scales, 1)


def _rms64(z):
    return 1.0 / ((z * z).sum(1, keepdim=True) / z.shape[1] + EPS).sqrt()


def _turn64(x, positions, freqs, factor, start, interleaved):
    n = freqs.shape[0]
    at = start + torch.arange(n, device=x.device)
    i, j = (start + 2 * (at - start), start + 2 * (at - start) + 1) if interleaved else (at, at + n)
    w = torch.polar(torch.full((positions.shape[0], n), factor, dtype=torch.float64, device=x.device),
                    torch.outer(positions.double(), freqs))[:, None]
    z = torch.complex(x[..., i], x[..., j]) * w
    y = x.clone()
    y[..., i], y[..., j] = z.real, z.imag
    return y


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        got, z = {}, s["x"].double()
        if case["residual"]:
            z = z + s["residual"].double()
            got["residual_out"] = z
            z = z.to(s["x"].dtype).double()        # the norm is of the stored residual
        t, r = z * s["weight"].double(), _rms64(z)
        if not case["fp8"]:
            return {**got, "out": t * r}
        codes, sc = _groups64(t, r, case["ue8m0"])
        return {**got, "codes": codes, "scales": sc}
    if kind == "linear":
        if case["quant"]:
            a, sc = _groups64(s["x"].double(), torch.ones_like(s["x"][:, :1], dtype=torch.float64), False)
        else:
            a, sc = s["a"].double(), s["a_scales"].double()
        N, K = s["w"].shape
        out = torch.zeros(a.shape[0], N, dtype=torch.float64, device=DEV)
        row = torch.arange(N, device=DEV) // GROUP
        for b, k in enumerate(range(0, K, GROUP)):       # a block of K at a time, scaled after its sum
            part = a[:, k:k + GROUP] @ s["w"][:, k:k + GROUP].double().t()
            out += part * sc[:, b:b + 1].double() * s["w_scales"].double()[row, b]
        return out
    if kind == "rope":
        return _turn64(s["x"].double(), s["positions"], s["freqs"], s["factor"], case["start"], case["interleaved"])
    z = s["kv"][:, :LAT].double()
    t, r = z * s["weight"].double(), _rms64(z)
    pe = _turn64(s["kv"][:, None, LAT:].double(), s["positions"], s["freqs"], s["factor"], 0, case["interleaved"])[:, 0]
    got = {n: v.to(torch.float64) for n, v in _rows(s["cache"]).items()}
    on = s["slots"] >= 0
    at = s["slots"][on]
    if case["row"] == 656:
        codes, sc = _groups64(t, r, False)
        new = {"codes": codes, "scales": sc, "rope": pe}
    else:
        new = {"codes": _code_values((torch.cat((t * r, pe), 1) / KV_SCALE).clamp(-E4M3_MAX, E4M3_MAX))}
    for n, v in new.items():
        got[n][at] = v[on]
    return got
