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


def peak_case(dtype, seqs, positions, new, gap, peak, kv_heads=1, group=4, dim=64, page=128):
    """One position whose score stands `gap` above all others, which are alike, and whose values are zero: the result is what the
    tail's weights make of its values.  Returns (call, reference in 64 bits, largest value)."""
    gen = generator(positions + new)
    pages = positions // page
    k = torch.zeros((seqs * pages, kv_heads, page, dim), device="cuda")
    v = torch.randint(1, 5, k.shape, generator=gen, device="cuda").float()
    first = torch.arange(seqs, device="cuda") * pages + peak // page
    k[first, :, peak % page, 0] = gap
    v[first, :, peak % page] = 0
    q = torch.zeros((seqs * new, kv_heads * group, dim), device="cuda")
    q[..., 0] = 1
    scales = dict(k_scales=torch.ones((seqs * pages, kv_heads), device="cuda"), v_scales=torch.ones((seqs * pages, kv_heads), device="cuda"))
    table = torch.arange(seqs * pages, device="cuda").int().view(seqs, pages)
    args = (q.bfloat16(), k.to(dtype), v.to(dtype), table, ints([positions] * seqs))
    seen = positions - new + 1 + torch.arange(new, device="cuda")
    tail = v.view(seqs, pages, kv_heads, page, dim).transpose(2, 3).reshape(seqs, positions, kv_heads, dim).double().cumsum(dim=1)[:, seen - 1]
    there = (seen > peak).double()[None, :, None, None]
    share = there * math.exp(-gap) + (1 - there)
    want = tail * share / (there + (seen[None, :, None, None] - there) * share)
    want = want.repeat_interleave(group, dim=2).reshape(q.shape)
    return args, scales if dtype == FP8 else {}, want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [15, 16, 18, 20])
@pytest.mark.parametrize("seqs,positions,new,kv_heads,peak", [(1, 65536, 1, 1, 77), (128, 4096, 1, 8, 1030), (128, 4096, 3, 8, 4090), (1, 65536, 512, 1, 65000),
                                                              (32, 4096, 64, 8, 5), (32, 4096, 64, 8, 3000)])
def test_a_peak_without_values_leaves_the_tail(dtype, gap, seqs, positions, new, kv_heads, peak):
    """Rounding of the result 2^-8 and of a weight 2^-8 (bf16 pages, more than 32 rows per KV head) or 2^-11, scores and sums 2^-14;
    E4M3 pages: an f16 weight loses at most half of 2^-24 below 2^11 times the largest, 2^-36 of the largest value a position."""
    from thor_megakernels_b200 import paged

    args, scales, want = peak_case(dtype, seqs, positions, new, gap, peak, kv_heads)
    got = paged.attention(*args, scale=1.0, **scales)
    paged.check_errors()
    many = dtype == torch.bfloat16 and new * 4 > 32
    tol = (2.0 ** -8 + (2.0 ** -8 if many else 2.0 ** -11) + 2.0 ** -14) * want + (positions * 2.0 ** -36 * 4 if dtype == FP8 else 0)
    off = (got.double() - want).abs()
    assert (off <= tol).all(), float((off / want).max())


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_with_idle_and_bad_positions_keeps_the_pages(dtype):
    """Position -1: an idle slot.  A position beyond the cache: reported, and otherwise as idle.  Neither stores a row nor moves a
    page's scale, and the sequences beside them get what they get without."""
    from test_gpu_paged_decoder import build
    from thor_megakernels_b200._lib import MegakernelError
    from thor_megakernels_b200.batched import BatchedDecoder
    from thor_megakernels_b200.paged import PagedKvCache

    model = build(batch=4)
    cache = PagedKvCache.for_model(model, 16, page_size=16, max_seqs=4, max_positions=64, dtype=dtype)
    dec = BatchedDecoder(model, 4, cache=cache)
    for b in range(4):
        cache.reserve(b, 40)
        dec.prefill(ints([3 + b, 50, 7, 11, 900 + b, 2, 31]), slot=b)
    tensors = [t for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]
    kept = [t.clone() for t in tensors]
    tokens = ints([5, 6, 7, 8])
    dec.step(tokens, ints([7, 7, 7, 7]))
    want = dec.logits[1].clone()
    dec.status()
    mine = cache.page_table[1, :3].long()
    for bad, reported in (([-1, 7, -1, -5], False), ([-1, 7, 64, -2 ** 31], True), ([2 ** 31 - 1, 7, -1, 100], True)):
        for t, k in zip(tensors, kept):
            t.copy_(k)
        dec.step(tokens, ints(bad))
        if reported:
            with pytest.raises(MegakernelError):
                dec.status()
        dec.status()
        assert torch.equal(dec.logits[1], want)
        assert torch.isfinite(dec.logits).all()
        for t, k in zip(tensors, kept):
            others = torch.ones(t.shape[1], dtype=torch.bool, device="cuda")
            others[mine] = False
            assert torch.equal(t[:, others].view(torch.uint8), k[:, others].view(torch.uint8))
    dec.close()


@pytest.mark.parametrize("new", [2, 5, 40])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinite_values_in_the_causal_edge(new, sign):
    """bf16: the rows that see an infinite value are infinite in its column, not NaN; the others do not know of it."""
    from thor_megakernels_b200 import paged

    gen = generator(2)
    k, v, _, _ = pool(torch.bfloat16, 8, 1, 32, 64, gen)
    for length in (new, 33, 100, 190):
        if length < new:
            continue
        w = v.clone()
        at = length - 2
        args = (ints([[6, 1, 4, 3, 0, 2]]), ints([length]))
        q = torch.randn((new, 4, 64), generator=gen, device="cuda").bfloat16()
        clean = paged.attention(q, k, v, *args)
        w[int(args[0][0, at // 32]), 0, at % 32, 7] = sign * math.inf
        got = paged.attention(q, k, w, *args)
        assert torch.equal(got[:-2], clean[:-2])
        assert (got[-2:, :, 7] == sign * math.inf).all()
        keep = torch.arange(64, device="cuda") != 7
        assert torch.equal(got[-2:][..., keep], clean[-2:][..., keep])
    paged.check_errors()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_rows_over_missing_pages_are_zero_whatever_the_queries_hold(dtype, new, what):
    from thor_megakernels_b200 import paged

    gen = generator(3)
    k, v, ks, vs = pool(dtype, 8, 1, 32, 64, gen)
    table, lengths = ints([[-1] * 6, [0, 1, 2, 3, 4, 5], [-1, -1, 6, 7, -1, -1]]), ints([150, 150, 150])
    q = torch.randn((3 * new, 4, 64), generator=gen, device="cuda").bfloat16()
    scales = dict(k_scales=ks, v_scales=vs)
    clean = paged.attention(q, k, v, table, lengths, **scales)
    q[:new] = what
    got = paged.attention(q, k, v, table, lengths, **scales)
    assert (got[:new] == 0).all() and torch.equal(got[new:], clean[new:])
    paged.check_errors()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,new", [(15, 10), (16, 9), (20, 3), (1000, 40), (0, 60), (19, 1), (20, 1)])
def test_rows_beyond_the_rotary_tables_are_left_out(dtype, start, new):
    """Tables of 20 positions: rows below are stored and rotated as if they came alone, those at or past the end are left out."""
    from thor_megakernels_b200 import paged
    from thor_megakernels_b200._lib import MegakernelError

    gen = generator(4)
    pages = 1200 // 16
    a, b = (pool(dtype, pages, 2, 16, 64, generator(5)) for _ in range(2))
    table = torch.arange(pages, device="cuda").int().view(1, pages)
    rows = [torch.randn((new, h, 64), generator=gen, device="cuda").bfloat16() for h in (2, 2, 4)]
    rows[0][-1] *= 1000   # would move a page's scale
    rows[1][-1] *= 1000
    angle = torch.rand((20, 32), generator=gen, device="cuda") * 6
    tables = dict(rope_cos=angle.cos(), rope_sin=angle.sin(), layout="half")
    outs = [torch.full_like(rows[2], 5.0) for _ in range(2)]
    paged.append(rows[0], rows[1], a[0], a[1], table, ints([start]), q=rows[2], q_out=outs[0], k_scales=a[2], v_scales=a[3], **tables)
    if start + new > 20:
        with pytest.raises(MegakernelError):
            paged.check_errors()
    fits = max(0, min(new, 20 - start))
    if fits:
        paged.append(rows[0][:fits], rows[1][:fits], b[0], b[1], table, ints([start]), q=rows[2][:fits], q_out=outs[1][:fits], k_scales=b[2],
                     v_scales=b[3], **tables)
    paged.check_errors()
    assert torch.equal(*outs)
    for x, y in zip(a, b):
        if x is not None:
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_reserve_and_release_do_not_wait_for_the_device():
    """The table changes behind what is queued, and the host goes on."""
    from thor_megakernels_b200 import paged

    cache = paged.PagedKvCache(1, 8, 1, 64, page_size=16, max_seqs=3, max_positions=64)
    cache.reserve(0, 5)   # the first pinned block is allocated
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(400_000_000)   # some 0.2 s of device time
    cache.reserve(1, 30)
    cache.reserve(2, 64)
    cache.release(1)
    cache.reserve(0, 40)
    done.record()
    assert not done.query()
    torch.cuda.synchronize()
    assert cache.page_table.tolist() == [[0, 1, 2, -1], [-1] * 4, [3, 4, 5, 6]]
    assert cache.free_pages == 1


def test_pages_are_not_handed_out_inside_a_capture():
    """The table would change with every replay and not now, the host's lists now and never again."""
    from thor_megakernels_b200 import paged

    cache = paged.PagedKvCache(1, 8, 1, 64, page_size=16, max_seqs=3, max_positions=64)
    cache.reserve(0, 40)
    before = cache.page_table.clone()
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="capture"):
            cache.reserve(1, 20)
        with pytest.raises(RuntimeError, match="capture"):
            cache.release(0)
    graph.replay()
    assert cache.free_pages == 5 and torch.equal(cache.page_table, before) and (x == 1).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_most_sequences_of_a_call(dtype):
    """1024 ragged sequences, a few of them prompts, D = 128: both kernels with their largest lists of sequences."""
    from thor_megakernels_b200 import paged

    gen = generator(6)
    seqs, page = 1024, 16
    new = [(0, 1, 3)[b % 3] if b % 128 != 5 else 40 for b in range(seqs)]
    lengths = [n + (7 * b) % 50 for b, n in enumerate(new)]
    k, v, ks, vs = pool(dtype, seqs * 6, 1, page, 128, gen)
    table = torch.randperm(seqs * 6, generator=gen, device="cuda").int().view(seqs, 6)
    cu = ints([0] + list(torch.tensor(new).cumsum(0)))
    q = torch.randn((sum(new), 2, 128), generator=gen, device="cuda").bfloat16()
    got = paged.attention(q, k, v, table, ints(lengths), k_scales=ks, v_scales=vs, cu_tokens=cu)
    paged.check_errors()
    kd, vd = po.dequantise(k, ks), po.dequantise(v, vs)
    want, mag = po.attention(q, kd, vd, table, ints(lengths), cu, page, 1 / math.sqrt(128))
    tol = po.attention_tolerance(want, mag, dtype == FP8, 90, float(vd.abs().max()), True)
    assert not torch.isnan(got).any() and ((got.double() - want).abs() <= tol).all()
    with pytest.raises(Exception, match="more sequences"):
        paged.attention(q, k, v, table.repeat(2, 1)[:1025], ints(lengths + [0]), k_scales=ks, v_scales=vs, cu_tokens=torch.cat((cu, cu[-1:])))
