"""Grids of 2^32 threads, which no launch takes, are refused as a limit by the dense attentions (on the CPU: before a launch)."""
import pytest

from arcagi2_flashnext_dots3_amd import _lib

LIMIT = -5


def prompt(B, T, H, D=64):
    return (256, 64, 64, 256, 64, 64, 256, 64, 64, 256, B, T, H, H, D, D, 1.0, 1, 2, 256, 64, 64, None, 0, None)


def chunk(B, T, H, row, W=5):
    return (256, 576, 576, 256, 80, row, 16, 16, 256, W, W, 256, 256, B, T, H, 1.0, 1.0, 16 * W, 0, 256, 512, 512, None, 0, None, 0, None)


@pytest.mark.parametrize("name,args", [
    ("spmla_attn_prompt", prompt(1 << 18, 1 << 18, 128)),              # 2^25 workgroups and more of 256 threads
    ("spmla_attn_prompt", prompt(1 << 20, 1 << 20, 128, 256)),
    ("spmla_attn_prompt", prompt(3, 1 << 22, 65536, 128)),             # of 512 threads
    ("spmla_attn_chunk", chunk(1 << 23, 1 << 23, 1, 656)),             # 2^23 of 512 threads
    ("spmla_attn_chunk", chunk(1 << 23, 1 << 23, 1, 576)),
    ("spmla_attn_chunk", chunk(3, 1 << 22, 65536, 576)),               # 2^31 of 256
])
def test_refused_before_a_launch(name, args):
    assert getattr(_lib.lib(), name)(*args) == LIMIT
