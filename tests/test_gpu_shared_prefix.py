"""Decode attention over shared prefixes against attention in 64 bits."""
import pytest
import torch

from shared_prefix_util import allowed, attend64, make_batch, on_device

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def run(b, device):
    from tinyvllm.kernels.shared_prefix import paged_decode_shared_prefix

    q, cache, meta, plan, out = on_device(b, device)
    paged_decode_shared_prefix(q, cache, 0, meta, plan, out, scale=b["scale"])
    torch.cuda.synchronize()
    return out


def check(b, out):
    want, mass, qk = attend64(b)
    err = (out.cpu().double() - want).abs()
    limit = allowed(b, want, mass, qk, out.dtype)
    assert torch.isfinite(out).all()
    assert (err <= limit).all(), f"{float((err / limit).max()):.2f} times the bound"


SHAPES = [  # heads, kv heads, dim, dtype, fp8, layout, block size
    (8, 8, 128, BF16, False, "token_major", 16),
    (32, 8, 128, BF16, False, "head_major", 16),
    (16, 2, 128, F16, False, "token_major", 16),
    (10, 2, 128, BF16, True, "token_major", 16),
    (12, 4, 64, F16, False, "head_major", 8),
    (8, 2, 64, BF16, True, "head_major", 1),
    (8, 2, 32, BF16, False, "token_major", 24),
    (6, 2, 32, F16, True, "token_major", 16),
    (8, 1, 256, BF16, False, "token_major", 32),
    (4, 2, 256, F16, True, "head_major", 256),
    (8, 2, 96, BF16, False, "token_major", 16),
    (40, 2, 80, F16, False, "token_major", 7),
    (9, 3, 8, BF16, False, "token_major", 16),
    (4, 2, 200, BF16, True, "token_major", 16),
    (150, 1, 128, BF16, False, "token_major", 16),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("count", [2, 5, 40])
def test_one_group(device, shape, count):
    """A group of rows behind one prefix of several tiles, own parts of every
    kind of end (none, one token, odd, several chunks), and rows apart."""
    heads, kv_heads, dim, dtype, fp8, layout, bs = shape
    prefix = -(-330 // bs) * bs
    own = [0, 1, 2, 17, 63, 64, 65, 130, 300]
    rows = [(0, own[i % len(own)]) for i in range(count)] + [(-1, 77), (-1, 0), (-1, 1)]
    b = make_batch(seed=count, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, fp8=fp8,
                   layout=layout, block_size=bs, prefixes=[prefix], rows=rows)
    out = run(b, device)
    assert (out[count + 1] == 0).all()
    check(b, out)
