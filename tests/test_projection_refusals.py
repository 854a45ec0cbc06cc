"""Arguments that the norm, quantization, projection, rotary and latent-row calls refuse, on the CPU: by the wrappers
(ValueError before the library) and by the library (its codes before a launch)."""
import pytest
import torch

from arcagi2_flashnext_dots3_amd import _lib, kernels, mla_fp8

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _refused(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def test_norm():
    x, w = _t(4, 256), _t(256)
    _refused("one GPU", kernels.rms_norm, x, w)                              # host tensors
    _refused("x \\[T, D\\]", kernels.rms_norm, x[0], w)
    _refused("x \\[T, D\\]", kernels.rms_norm, x.to(torch.float64), w)
    _refused("D > 0", kernels.rms_norm, _t(4, 0), None)
    _refused("contiguous rows", kernels.rms_norm, _t(4, 512)[:, ::2], w)
    _refused("weight", kernels.rms_norm, x, _t(255))
    _refused("weight", kernels.rms_norm, x, w.to(torch.float16))
    _refused("residual \\[T, D\\]", kernels.rms_norm, x, w, residual=_t(3, 256))
    _refused("residual \\[T, D\\]", kernels.rms_norm, x, w, residual=x.float())
    _refused("without a residual", kernels.rms_norm, x, w, residual_out=_t(4, 256))
    _refused("overlap", kernels.rms_norm, x, w, residual=_t(1, 256).expand(4, 256))
    _refused("overlap", kernels.rms_norm, x, w, out=_t(1, 256).expand(4, 256))
    _refused("out", kernels.rms_norm, x, w, out=x.float())
    _refused("codes", kernels.rms_norm_fp8, x, w, codes=_t(4, 256, dtype=torch.int8))
    _refused("scales", kernels.rms_norm_fp8, x, w, scales=_t(4, 1, dtype=torch.float32))
    _refused("x \\[T, D\\]", kernels.quant_fp8, _t(2, 3, 4))
    _refused("scales", kernels.quant_fp8, x, scales=_t(4, 2, dtype=BF))


def test_linear():
    a, w = _t(4, 256, dtype=F8), _t(300, 256, dtype=F8)
    sa, sw = _t(4, 2, dtype=torch.float32), _t(3, 2, dtype=torch.float32)
    _refused("one GPU", kernels.linear_fp8, a, sa, w, sw)
    _refused("a \\[T, K\\], w", kernels.linear_fp8, a, sa, w[:, :128], sw)
    _refused("multiple of 16", kernels.linear_fp8, a[:, :120], sa, w[:, :120], sw)
    _refused("multiple of 16", kernels.linear_fp8, a[:, :0], sa, w[:, :0], sw)
    _refused("a \\[T, K\\] e4m3", kernels.linear_fp8, _t(4, 256), sa, w, sw)
    _refused("w \\[N, K\\] e4m3", kernels.linear_fp8, a, sa, _t(300, 512, dtype=F8)[:, ::2], sw)
    _refused("a_scales", kernels.linear_fp8, a, sa[:, :1], w, sw)
    _refused("w_scales", kernels.linear_fp8, a, sa, w, sw[:2])
    _refused("w_scales", kernels.linear_fp8, a, sa, w, sw.double())
    _refused("out", kernels.linear_fp8, a, sa, w, sw, dtype=torch.float32)
    _refused("out", kernels.linear_fp8, a, sa, w, sw, out=_t(4, 299))
    _refused("overlap", kernels.linear_fp8, a, sa, w, sw, out=_t(1, 300).expand(4, 300))
    _refused("bf16 / fp16", mla_fp8.linear_fp8, _t(4, 256, dtype=torch.float32), (w, sw))


def test_linear_quant():
    x, w, sw = _t(4, 256), _t(300, 256, dtype=F8), _t(3, 2, dtype=torch.float32)
    _refused("one GPU", kernels.linear_quant, x, w, sw)
    _refused("x \\[T, K\\], w", kernels.linear_quant, x, w[:, :128], sw)
    _refused("multiple of 16", kernels.linear_quant, x[:, :120], w[:, :120], sw)
    _refused("D > 0", kernels.linear_quant, x[:, :0], w[:, :0], sw)
    _refused("x \\[T, D\\]", kernels.linear_quant, x.to(F8), w, sw)
    _refused("w \\[N, K\\] e4m3", kernels.linear_quant, x, _t(300, 256), sw)
    _refused("w_scales", kernels.linear_quant, x, w, sw[:, :1])
    _refused("out", kernels.linear_quant, x, w, sw, out=_t(4, 299))
    _refused("out", kernels.linear_quant, x, w, sw, out=_t(4, 300, dtype=torch.float32))
    _refused("overlap", kernels.linear_quant, x, w, sw, out=_t(1, 300).expand(4, 300))
    _refused("unpack", kernels.linear_quant, x[0], w, sw)


def test_rope():
    x, pos, f = _t(4, 2, 64), torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    _refused("one GPU", kernels.rope, x, pos, f)
    _refused("x \\[T, H, W\\]", kernels.rope, x.to(torch.float64), pos, f)
    _refused("positions", kernels.rope, x, pos[:3], f)
    _refused("positions", kernels.rope, x, pos.float(), f)
    _refused("freqs", kernels.rope, x, pos, f.float())
    _refused("inside the head", kernels.rope, x, pos, f, start=1)
    _refused("inside the head", kernels.rope, x, pos, f[:8], start=-1)
    _refused("out of x's", kernels.rope, x, pos, f, out=x.float())
    _refused("contiguous head", kernels.rope, _t(4, 2, 128)[..., ::2], pos, f)
    _refused("overlap", kernels.rope, x, pos, f, out=_t(4, 1, 64).expand(4, 2, 64))
    _refused("overlap", kernels.rope, x, pos, f, out=_t(5 * 64).as_strided((4, 2, 64), (64, 64, 1)))
    _refused("overlap", kernels.rope, x, pos, f, out=_t(1024).as_strided((4, 2, 64), (65, 64, 1)))
    _refused("one GPU", kernels.rope, x, pos, f, out=_t(2, 4, 64).transpose(0, 1))       # heads outermost: taken


def test_latent_write():
    kv, w = _t(4, 576), _t(512)
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    slots, cache = torch.arange(4), _t(8, 656, dtype=torch.uint8)
    args = (kv, w, 1e-6, pos, f, slots, cache)
    _refused("one GPU", kernels.latent_write, *args)
    _refused("kv", kernels.latent_write, kv[:, :575], *args[1:])
    _refused("weight", kernels.latent_write, kv, w[:511], *args[2:])
    _refused("positions", kernels.latent_write, kv, w, 1e-6, pos[:3], f, slots, cache)
    _refused("freqs", kernels.latent_write, kv, w, 1e-6, pos, f[:16], slots, cache)
    _refused("slots", kernels.latent_write, kv, w, 1e-6, pos, f, slots.to(torch.int32), cache)
    _refused("cache rows", kernels.latent_write, *args, fmt=1)
    _refused("fmt", kernels.latent_write, *args, fmt=3)


@pytest.mark.parametrize("name,args,code", [
    # (256, 264 ...: placeholder addresses that the checks reject before anything is launched)
    ("spmla_rms_norm", (256, 8, None, 0, None, 0, None, 0, 1e-6, -1, 8, 2, 256, 8, None, 0, None, 0, 0, None), -2),
    ("spmla_rms_norm", (256, 8, None, 0, None, 0, None, 0, 1e-6, 1, 0, 2, 256, 8, None, 0, None, 0, 0, None), -2),
    ("spmla_rms_norm", (256, 8, None, 0, None, 0, None, 0, -1.0, 1, 8, 2, 256, 8, None, 0, None, 0, 0, None), -2),
    ("spmla_rms_norm", (256, 8, None, 0, None, 0, None, 0, 1e-6, 1, 8, 3, 256, 8, None, 0, None, 0, 0, None), -2),
    ("spmla_rms_norm", (256, 8, None, 0, None, 0, None, 0, 1e-6, 1, 8, 2, None, 8, None, 0, None, 0, 0, None), -2),
    ("spmla_rms_norm", (256, 8, 256, 8, None, 0, None, 0, 1e-6, 1, 8, 2, 256, 8, None, 0, None, 0, 0, None), -2),
    ("spmla_rms_norm", (256, 8, None, 0, None, 0, None, 0, 1e-6, 1, 8, 2, None, 8, 256, 8, None, 0, 0, None), -2),
    ("spmla_rms_norm", (256, 1 << 17, None, 0, None, 0, None, 0, 1e-6, 1, 65537, 2, 256, 1 << 17, None, 0, None, 0, 0, None), -5),
    ("spmla_rms_norm", (257, 8, None, 0, None, 0, None, 0, 1e-6, 1, 8, 2, 256, 8, None, 0, None, 0, 0, None), -3),
    ("spmla_quant_fp8", (256, 8, 1, 0, 2, 256, 8, 256, 1, 0, None), -2),
    ("spmla_quant_fp8", (256, 8, 1, 8, 2, None, 8, 256, 1, 0, None), -2),
    ("spmla_quant_fp8", (256, 8, 1, 8, 2, 256, 8, 258, 1, 0, None), -3),
    ("spmla_linear_fp8", (256, 32, 256, 1, 256, 32, 256, 1, 1, 8, 24, 2, 256, 8, None), -2),          # K % 16
    ("spmla_linear_fp8", (256, 32, 256, 1, 256, 32, 256, 1, 1, 8, 32, 0, 256, 8, None), -2),          # fp32 output
    ("spmla_linear_fp8", (256, 16, 256, 1, 256, 32, 256, 1, 2, 8, 32, 2, 256, 8, None), -2),          # rows overlap
    ("spmla_linear_fp8", (264, 32, 256, 1, 256, 32, 256, 1, 1, 8, 32, 2, 256, 8, None), -3),
    ("spmla_linear_fp8", (256, 40, 256, 1, 256, 32, 256, 1, 2, 8, 32, 2, 256, 8, None), -3),
    ("spmla_linear_fp8", (256, 1 << 23, 256, 1, 256, 32, 256, 1, 2, 8, 32, 2, 256, 8, None), -5),
    ("spmla_linear_fp8", (None, 32, 256, 1, 256, 32, 256, 1, 1, 8, 32, 2, 256, 8, None), -2),
    ("spmla_rope", (256, 64, 64, 256, 0, 256, 1, 1, 64, 2, 32, 1, 1.0, 0, 2, 512, 64, 64, None), -2),   # past the head
    ("spmla_rope", (256, 64, 64, 256, 0, 256, 1, 1, 64, 0, 32, 1, 1.0, 0, 2, 256, 128, 64, None), -2),  # in place, strides
    ("spmla_rope", (256, 64, 64, None, 0, 256, 1, 1, 64, 0, 32, 1, 1.0, 0, 2, 512, 64, 64, None), -2),
    ("spmla_rope", (257, 64, 64, 256, 0, 256, 1, 1, 64, 0, 32, 1, 1.0, 0, 2, 512, 64, 64, None), -3),
    ("spmla_rms_norm", (256, 8, None, 0, None, 0, None, 0, 1e-6, (1 << 23) + 1, 8, 2, 256, 8, None, 0, None, 0, 0, None), -5),
    ("spmla_quant_fp8", (256, 8, (1 << 23) + 1, 8, 2, 256, 8, 256, 1, 0, None), -5),
    ("spmla_linear_fp8", (256, 32, 256, 1, 256, 32, 256, 1, (1 << 23) + 1, 8, 32, 2, 256, 8, None), -5),
    ("spmla_linear_fp8", (256, 32, 256, 1, 256, 32, 256, 1, 1 << 23, 1 << 23, 32, 2, 256, 1 << 23, None), -5),   # too many tiles
    ("spmla_rope", (256, 64, 64, 256, 0, 256, (1 << 23) + 1, 1, 64, 0, 32, 1, 1.0, 0, 2, 512, 64, 64, None), -5),
    ("spmla_latent_write", (256, 576, None, 0, 1e-6, 256, 0, 256, 1, 1.0, 256, (1 << 23) + 1, 256, 8, 8, 8 * 656, 0, 1.0, None), -5),
    ("spmla_latent_write", (256, 576, None, 0, 1e-6, 256, 0, 256, 1, 1.0, 256, 1, 256, 8, 8, 8 * 656, 3, 1.0, None), -2),
    ("spmla_latent_write", (256, 576, None, 0, 1e-6, 256, 0, 256, 1, 1.0, 256, 1, 256, 8, 8, 8 * 576, 1, 0.0, None), -2),
    ("spmla_latent_write", (258, 576, None, 0, 1e-6, 256, 0, 256, 1, 1.0, 256, 1, 256, 8, 8, 8 * 656, 0, 1.0, None), -3),
    ("spmla_latent_write", (256, 576, None, 0, 1e-6, 256, 0, 256, 1, 1.0, 256, 1, 256, 8, 8, 8, 0, 1.0, None), -3),
])
def test_codes_before_a_launch(name, args, code):
    assert _lib.status(name, *args) == code
