"""MLA's absorbed per-head matmuls on FP8 weights: the reference's mla_fp8 (dotsnote/engine/arcstats_pkg/arcstats/
mla_fp8.py) and the in-place decode query build of qcat.py, on libspmla_gfx950.so.

kv_b_proj is block-FP8 in the checkpoint (128 x 128 blocks, weight_scale_inv); vLLM's bf16 W_UK_T / W_UV are
round_bf16(code * scale). convert() recovers the codes exactly (checked bit for bit after the round trip, mla_fp8.py:
89-94) so the kernels read half the weight bytes and dequantize to the same bf16 values in registers.

linear_fp8() is the layer's plain projections (down, up, output) on the checkpoint's codes and block scales, with the
activations in 8 bits too.
"""
import torch

from . import kernels


def codes_of(wbf, scale_full):
    """wbf bf16 weight, scale_full fp32 of the same shape -> e4m3 codes (uint8), or None unless every element comes back
    bit for bit as bf16(code * scale) (the exactness rule of mla_fp8.py:89-94)."""
    codes = (wbf.float() / scale_full).to(torch.float8_e4m3fn)
    again = (codes.float() * scale_full).to(torch.bfloat16)
    if not torch.equal(again.view(torch.int16), wbf.view(torch.int16)):
        return None
    return codes.view(torch.uint8)


def convert(W_UK_T, W_UV, weight_scale_inv):
    """W_UK_T [N, P, L], W_UV [N, L, V] bf16 and kv_b_proj's block scales [(N (P + V)) / 128, L / 128] -> the FP8
    forms (uk, uv) of mla_fp8._convert (:97-139): uk = (codes [N, L, P], scales [N, P, L / 128], scale_k False),
    uv = (codes [N, V, L], scales [N, V, L / 128], scale_k True); None when a round trip is not exact.
    kv_b_proj's rows are head-major, each head's P key rows before its V value rows; a 128 x 128 block scale covers
    128 consecutive rows and 128 columns."""
    N, P, L = W_UK_T.shape
    V = W_UV.shape[2]
    blocks = weight_scale_inv.float()
    if blocks.dim() != 2 or blocks.shape[0] != (N * (P + V) + 127) // 128 or blocks.shape[1] != (L + 127) // 128:
        return None
    per_row = blocks.repeat_interleave(128, dim=0)[: N * (P + V)].view(N, P + V, blocks.shape[1])
    key_scales, value_scales = per_row[:, :P], per_row[:, P:]          # [N, P, L / 128], [N, V, L / 128]
    per_col = lambda sc: sc.repeat_interleave(128, dim=2)[..., :L]   # one scale per element
    c_uk = codes_of(W_UK_T, per_col(key_scales))
    c_uv = codes_of(W_UV.transpose(1, 2), per_col(value_scales))
    if c_uk is None or c_uv is None:
        return None
    return ((c_uk.transpose(1, 2).contiguous(), key_scales.contiguous(), False),
            (c_uv.contiguous(), value_scales.contiguous(), True))


def bmm_fp8(a, f, out=None):
    """a [N, B, K] bf16 (any strides), f = (codes [N, J, K], scales, scale_k) -> out [N, B, J] (mla_fp8.bmm_fp8)."""
    codes, scales, scale_k = f
    if out is None:
        out = torch.empty((a.shape[0], a.shape[1], codes.shape[1]), dtype=a.dtype, device=a.device)
    return kernels.bmm_fp8(a, codes, scales, scale_k, out)


def linear_fp8(x, f, out=None, ue8m0=False):
    """x [T, K] bf16 / fp16, quantized here per 128 values (kernels.quant_fp8), or (codes, scales) from
    kernels.rms_norm_fp8 / quant_fp8; f = (weight codes [N, K] e4m3, weight_scale_inv [ceil(N / 128), ceil(K / 128)])
    -> out [T, N] in x's type (bf16 for codes)."""
    codes, scales = f
    if isinstance(x, torch.Tensor):
        if x.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("linear_fp8: x bf16 / fp16, or (codes, scales)")
        return kernels.linear_quant(x, codes, scales, out=out, ue8m0=ue8m0)
    a, sa = x
    return kernels.linear_fp8(a, sa, codes, scales, out=out)


def build_query(q_nope, q_pe, f_uk, out=None):
    """The concatenated decode query [T, H, 576] = (q_nope @ W_UK_T, q_pe) in one launch (qcat.py: the bmm writes
    the first 512 columns in place, q_pe fills the rest). q_nope [T, H, 128], q_pe [T, H, 64] bf16."""
    codes, scales, scale_k = f_uk
    if scale_k or tuple(codes.shape[1:]) != (512, 128):
        raise ValueError("build_query: f_uk must be convert()'s W_UK_T form (codes [H, 512, 128])")
    return kernels.mla_query(q_nope, q_pe, codes, scales, out)
