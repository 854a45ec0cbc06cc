"""Values, alignments and limits that the norm, projection, rotary and latent-row calls refuse: ValueError with the argument's
name, before anything is launched (the device is looked at last: host tensors that pass reach that check)."""
import pytest
import torch

from arcagi2_flashnext_dots3_amd import _lib, kernels

BF, F8, F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32


def _refused(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def _at(shape, dtype, offset, pitch=None):
    """Zeros of `shape` that begin `offset` elements into an aligned buffer, rows `pitch` elements apart."""
    pitch = pitch or shape[-1]
    return torch.zeros(shape[0] * pitch + offset + 64, dtype=dtype).as_strided(shape, (pitch, 1), offset)


def test_norm_and_quantization():
    x = torch.zeros(2, 256, dtype=BF)
    for eps in (-1e-6, float("nan")):
        _refused("eps", kernels.rms_norm, x, None, eps)
    _refused("D of 65544", kernels.rms_norm, torch.zeros(1, 65544, dtype=BF), None)
    _refused("T of 8388609", kernels.rms_norm, torch.zeros((1 << 23) + 1, 1, dtype=BF), None)
    _refused("T of 8388609", kernels.quant_fp8, torch.zeros((1 << 23) + 1, 1, dtype=BF))
    _refused("one GPU", kernels.rms_norm, _at((2, 256), BF, 3, 259), None)              # any alignment is taken


def _product(T=4, N=300, K=272):
    return [torch.zeros(T, K, dtype=F8), torch.zeros(T, 3), torch.zeros(N, K, dtype=F8), torch.zeros(-(-N // 128), 3)]


@pytest.mark.parametrize("quant", [False, True])
def test_weights_of_a_projection(quant):
    def call(w, sw, T=4, K=272, **kw):
        if quant:
            return kernels.linear_quant(torch.zeros(T, K, dtype=BF), w, sw, **kw)
        return kernels.linear_fp8(torch.zeros(T, K, dtype=F8), torch.zeros(T, -(-K // 128)), w, sw, **kw)
    _, _, w, sw = _product()
    _refused("one GPU", call, w, sw)
    _refused("w .*rows on 16 bytes", call, _at((300, 272), F8, 8), sw)
    _refused("w .*rows on 16 bytes", call, _at((300, 272), F8, 0, 280), sw)
    _refused("w .*overlap", call, w[:1].expand(300, 272), sw)
    _refused("w_scales .*overlap", call, w, sw[:1].expand(3, 3))
    _refused("stride of w of", call, _at((2, 272), F8, 0, (1 << 22) + 16), sw[:1])
    _refused("K of", call, torch.zeros(1, (1 << 22) + 16, dtype=F8), torch.zeros(1, 32769), T=1, K=(1 << 22) + 16)
    _refused("N of", call, torch.zeros((1 << 23) + 16, 16, dtype=F8), torch.zeros(65537, 1), T=1, K=16)
    _refused("one GPU", call, _at((300, 272), F8, 8), sw, T=0)                          # nothing to read


def test_activations_of_a_projection():
    a, sa, w, sw = _product()
    _refused("a .*rows on 16 bytes", kernels.linear_fp8, _at((4, 272), F8, 4), sa, w, sw)
    _refused("a .*rows on 16 bytes", kernels.linear_fp8, _at((4, 272), F8, 0, 274), sa, w, sw)
    _refused("a .*overlap", kernels.linear_fp8, a[:1].expand(4, 272), sa, w, sw)
    _refused("a_scales .*overlap", kernels.linear_fp8, a, sa[:1].expand(4, 3), w, sw)
    _refused("stride of a of", kernels.linear_fp8, _at((2, 272), F8, 0, (1 << 22) + 16), sa[:2], w, sw)
    _refused("stride of a_scales", kernels.linear_fp8, a[:2], _at((2, 3), F32, 0, (1 << 20) + 1), w, sw)
    _refused("one GPU", kernels.linear_fp8, torch.zeros(272, 1, dtype=F8).t(), sa[:1], w, sw)   # a single row: any stride


def test_tiles_of_a_projection():
    """More tiles than a grid holds, whichever kernel: named before the output is looked at."""
    n = 1 << 23
    a, s = torch.zeros(n, 16, dtype=F8), torch.zeros(n, 1)
    _refused("more tiles", kernels.linear_fp8, a, s, a, s[:65536], out=s)
    assert _lib.status("spmla_linear_fp8", 256, 16, 256, 1, 256, 16, 256, 1, n, n, 16, 2, 256, n, None) == -5


def test_rotary():
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(8, dtype=torch.float64)
    b = torch.zeros(512)
    x = b.as_strided((4, 2, 16), (32, 16, 1))
    _refused("x's strides", kernels.rope, x, pos, f, out=b.as_strided((4, 2, 16), (64, 16, 1)))
    _refused("x's strides", kernels.rope, x, pos, f, out=b.as_strided((4, 2, 16), (16, 64, 1)))
    _refused("one GPU", kernels.rope, x[:1], pos[:1], f, out=b.as_strided((1, 2, 16), (64, 16, 1)))
    _refused("T of 8388609", kernels.rope, torch.zeros((1 << 23) + 1, 2, dtype=BF), torch.zeros((1 << 23) + 1, dtype=torch.int32), f[:1])


def test_latents():
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    slots, cache = torch.arange(4), torch.zeros(8, 656, dtype=torch.uint8)
    kv, w = torch.zeros(4, 576, dtype=BF), torch.zeros(512, dtype=BF)

    def call(kv=kv, w=w, eps=1e-6, cache=cache, **kw):
        kernels.latent_write(kv, w, eps, pos, f, slots, cache, **kw)
    _refused("one GPU", call)
    _refused("eps", call, eps=-1.0)
    _refused("kv .*rows on 16 bytes", call, kv=_at((4, 576), BF, 4))
    _refused("kv .*rows on 16 bytes", call, kv=_at((4, 576), BF, 0, 580))
    _refused("weight .*rows on 16 bytes", call, w=torch.zeros(516, dtype=BF)[4:])
    _refused("cache.* 8 bytes", call, cache=torch.zeros(8 * 656 + 8, dtype=torch.uint8)[4:-4].view(8, 656))
    _refused("cache.* 8 bytes", call, cache=torch.zeros(3000, dtype=torch.uint8).as_strided((2, 2, 656), (1316, 656, 1)))
    _refused("overlap", call, cache=torch.zeros(3000, dtype=torch.uint8).as_strided((2, 2, 656), (656, 656, 1)))
    _refused("block_size", call, block_size=0)
    _refused("block_size", call, block_size=-4)
    for scale in (0.0, -1.0, float("nan"), 1e-60):
        _refused("kv_scale", call, cache=torch.zeros(8, 576, dtype=torch.uint8), fmt=1, kv_scale=scale)
    _refused("one GPU", call, kv=kv[:0], w=torch.zeros(516, dtype=BF)[4:])              # nothing to read


def test_codes_of_the_library_are_value_errors(monkeypatch):
    """What only an entry point's own checks refuse has been refused before a launch too."""
    for code, match in ((-2, "rope: bad argument"), (-3, "misaligned"), (-5, "limit")):
        monkeypatch.setattr(_lib, "_TENSOR_FN", {"rope": lambda *a: code})
        _refused(match, _lib.tensor_call, "rope", None)
    monkeypatch.setattr(_lib, "_TENSOR_FN", {"rope": lambda *a: 100})
    with pytest.raises(RuntimeError, match="hip error"):
        _lib.tensor_call("rope", None)


@pytest.mark.parametrize("fmt,rowb", [(0, 656), (1, 576), (2, 400)])
def test_latents_into_blocks_behind_the_caches_memory(fmt, rowb):
    """A [R, row] cache with a block_stride: the last block has to lie inside the memory that the tensor is part of."""
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    pool = torch.zeros(3 * (4 * rowb + 64) + rowb, dtype=torch.uint8)
    args = torch.zeros(4, 576, dtype=BF), None, 1e-6, pos, f, torch.arange(4)

    def call(R, at=0, **kw):
        kernels.latent_write(*args, pool[at:].as_strided((R, rowb), (rowb, 1)), fmt=fmt, **kw)
    apart = dict(block_size=4, block_stride=4 * rowb + 64)
    _refused("one GPU", call, 12, **apart)
    _refused("one GPU", call, 13, **apart)                    # one row in the fourth block
    _refused("behind its memory", call, 13, at=8, **apart)
    _refused("behind its memory", call, 12, block_size=4, block_stride=6 * rowb)
    for stride in (1 << 40, 1 << 62):
        _refused("behind its memory", call, 8, block_size=1, block_stride=stride)
    _refused("one GPU", call, 12, block_size=5)
    _refused("one GPU", call, 12)
