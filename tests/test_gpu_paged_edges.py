"""Paged cache, calls at the edges of what the documentation allows: many short segments per CTA, values that are not finite
where only some rows see them, positions beyond the tables, pages that are not there."""
import math

import pytest
import torch

import paged_oracle as po

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
DTYPES = [torch.bfloat16, FP8]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def pool(dtype, pages, heads, page, dim, gen):
    """(k, v, k_scales, v_scales): random pages."""
    out = []
    for _ in range(2):
        x = torch.randn((pages, heads, page, dim), generator=gen, device="cuda")
        if dtype == torch.bfloat16:
            out.append((x.bfloat16(), None))
        else:
            scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(2, 3)) / 448.0)))
            out.append(((x / scale[:, :, None, None]).clamp(-448, 448).to(dtype), scale))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [60, 33])
def test_nan_in_the_causal_edge_of_many_short_prompts(dtype, tokens):
    """96 prompts x 8 KV heads of one tile each, five or more per CTA one behind the other: the rows from a NaN value's position on
    have NaN in its column and no other row or column has, call after call."""
    from thor_megakernels_b200 import paged

    gen = generator(1)
    seqs, kv_heads, group, dim, page = 96, 8, 4, 64, 64
    k, v, ks, vs = pool(dtype, seqs, kv_heads, page, dim, gen)
    q = torch.randn((seqs * tokens, kv_heads * group, dim), generator=gen, device="cuda").bfloat16()
    args = (ints([[b] for b in range(seqs)]), ints([tokens] * seqs))
    scales = dict(k_scales=ks, v_scales=vs)
    clean = paged.attention(q, k, v, *args, **scales)
    assert torch.isfinite(clean).all()
    expect = torch.zeros((seqs, tokens, kv_heads, group, dim), dtype=torch.bool, device="cuda")
    nan = torch.tensor(math.nan, device="cuda").to(dtype)
    for b in range(seqs):
        for h in range(kv_heads):
            if (b + h) % 5 == 4:
                continue   # some segments without
            at, column = (7 * b + 11 * h) % tokens, (13 * b + 29 * h) % dim
            v[b, h, at, column] = nan
            expect[b, at:, h, :, column] = True
    expect = expect.view(clean.shape)
    for _ in range(20):
        got = paged.attention(q, k, v, *args, **scales)
        assert torch.equal(torch.isnan(got), expect)
        assert torch.equal(got[~expect], clean[~expect])
    paged.check_errors()
