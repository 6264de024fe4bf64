"""Append to and attention over a paged cache, bf16 and E4M3, against 64-bit restatements (paged_oracle.py)."""
import math

import pytest
import torch

import paged_oracle as po

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
DTYPES = [torch.bfloat16, FP8]


def pool(dtype, pages, heads, page, dim, gen, spread=1.0):
    """(k, v, k_scales, v_scales): random pages with a magnitude of their own per page and head."""
    out = []
    for _ in range(2):
        x = torch.randn((pages, heads, page, dim), generator=gen, device="cuda")
        x *= torch.exp2(spread * torch.randn((pages, heads, 1, 1), generator=gen, device="cuda"))
        if dtype == torch.bfloat16:
            out.append((x.bfloat16(), None))
        else:
            amax = x.abs().amax(dim=(2, 3)).double()
            scale = torch.exp2(torch.ceil(torch.log2(amax / 448.0))).float()
            out.append(((x / scale[:, :, None, None]).clamp(-448, 448).to(dtype), scale))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def page_table(lengths, page, pages, gen, extra_columns=0):
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full((len(lengths), max(need) + extra_columns), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    assert at <= pages
    return table


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check_attention(got, q, k, v, ks, vs, table, lengths, cu, page, scale):
    kd, vd = po.dequantise(k, ks), po.dequantise(v, vs)
    want, mag = po.attention(q, kd, vd, table, lengths, cu, page, scale)
    used = ~torch.isnan(want).all(dim=2)
    counts = [r1 - r0 for r0, r1 in (po.rows_of(cu, table.shape[0], q.shape[0], b) for b in range(table.shape[0]))]
    many = max(counts) * (q.shape[1] // k.shape[1]) > 32
    tol = po.attention_tolerance(want, mag, ks is not None, int(lengths.max()), float(vd[torch.isfinite(vd)].abs().max()), many)
    assert used.any()
    off = (got.double() - want).abs() - tol
    assert not torch.isnan(off[used]).any()
    assert float(off[used].max()) <= 0, float(off[used].max())


# --------------------------------------------------------------------------- append

def run_append(dtype, dim, page, layout, rot, new, start, heads=8, kv_heads=2, ragged=True, seed=0, panel=True):
    from thor_megakernels_b200 import paged

    gen = generator(seed)
    lengths = [max(0, s) + n for s, n in zip(start, new)]
    pages = sum(-(-n // page) for n in lengths) + 2
    k, v, ks, vs = pool(dtype, pages, kv_heads, page, dim, gen)
    table = page_table(lengths, page, pages, gen)
    tokens = sum(new)
    cu = ints([0] + list(torch.tensor(new).cumsum(0))) if ragged else None
    x = (torch.randn((tokens, (heads + 2 * kv_heads) * dim), generator=gen, device="cuda") * 2).bfloat16()
    parts = x.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1)
    q, kn, vn = (t.unflatten(1, (-1, dim)) if panel else t.unflatten(1, (-1, dim)).contiguous() for t in parts)
    positions = max(lengths) + 3
    angle = torch.rand((positions, rot), generator=gen, device="cuda") * 6.28 if rot else None   # no column relation: every column counts
    cos, sin = (angle.cos(), (angle * 1.3).sin()) if rot else (None, None)
    before = [t.clone() if t is not None else None for t in (k, v, ks, vs)]
    q_out = torch.full((tokens, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    got = paged.append(kn, vn, k, v, table, ints(start), q=q, q_out=q_out, rope_cos=cos, rope_sin=sin, layout=layout, k_scales=ks,
                       v_scales=vs, cu_tokens=cu)
    assert got is q_out
    paged.check_errors()

    def turned(t, row, s):
        t = t[row[0]:row[1]].double()
        if not rot:
            return t, t.abs()
        return po.rotate(t, cos[s:s + t.shape[0]].double(), sin[s:s + t.shape[0]].double(), layout)

    for b, (n, s) in enumerate(zip(new, start)):
        row = po.rows_of(cu, len(new), tokens, b)
        if s < 0:
            assert (q_out[row[0]:row[1]] == 7.0).all()
            continue
        want, mag = turned(q, row, s)
        assert ((q_out[row[0]:row[1]].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * mag).all()
    untouched = torch.ones((pages, page), dtype=torch.bool, device="cuda")
    for (now, old, scale, old_scale, source, is_k) in ((k, before[0], ks, before[2], kn, True), (v, before[1], vs, before[3], vn, False)):
        fresh = torch.zeros(pages, dtype=torch.bool, device="cuda")
        for b, (n, s) in enumerate(zip(new, start)):
            row = po.rows_of(cu, len(new), tokens, b)
            if s < 0 or n == 0:
                continue
            want, mag = turned(source, row, s) if is_k else (source[row[0]:row[1]].double(),) * 2
            for first in range(s - s % page, s + n, page):
                lo, hi = max(s, first), min(s + n, first + page)
                to, held = int(table[b, first // page]), lo - first
                w, m = want[lo - s:hi - s].transpose(0, 1), mag[lo - s:hi - s].transpose(0, 1).abs()
                untouched[to, held:hi - first] = False
                here = now[to, :, held:hi - first].double()
                if scale is None:
                    assert ((here - w).abs() <= (2.0 ** -8 * w.abs() + 2.0 ** -22 * m)).all()
                    continue
                fresh[to] = True
                for h in range(kv_heads):
                    amax = float(w[h].abs().max().float())
                    need = po.scale_for(amax)
                    expect = max(float(old_scale[to, h]), need) if held else need
                    sc = float(scale[to, h])
                    assert sc == expect, (sc, expect, amax)
                    err = (here[h] * sc - w[h]).abs()
                    assert (err <= 2.0 ** -4 * w[h].abs() + sc * 2.0 ** -10 + 2.0 ** -22 * m[h]).all()
                    if held:   # recoded by a power of two: exact down to the subnormals
                        a = now[to, h, :held].double() * sc
                        c = old[to, h, :held].double() * float(old_scale[to, h])
                        assert ((a - c).abs() <= sc * 2.0 ** -10).all()
                        normal = c.abs() >= sc * 2.0 ** -6
                        assert torch.equal(a[normal], c[normal])
                        untouched[to, :held] = False
        if scale is not None:
            assert torch.equal(scale[~fresh], old_scale[~fresh])
            same = now.view(torch.uint8).transpose(1, 2)[untouched] == old.view(torch.uint8).transpose(1, 2)[untouched]
        else:
            same = now.view(torch.int16).transpose(1, 2)[untouched] == old.view(torch.int16).transpose(1, 2)[untouched]
        assert same.all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page,layout,rot", [(64, 16, "interleaved", 64), (64, 128, "half", 32), (128, 32, "half", 128),
                                                 (128, 128, "interleaved", 16), (128, 64, "half", 96), (64, 32, "half", 0)])
def test_append_ragged(dtype, dim, page, layout, rot):
    run_append(dtype, dim, page, layout, rot, new=[1, 0, 37, 2 * page + 5, 3, page], start=[0, 5, page - 1, 3, page + 7, 2 * page], seed=dim + page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page,seqs,new", [(128, 64, 1, 1), (64, 16, 40, 1), (128, 16, 70, 3), (64, 64, 3, 200)])
def test_append_uniform_with_idle_sequences(dtype, dim, page, seqs, new):
    start = [(17 * b) % 150 if b % 5 != 3 else -1 for b in range(seqs)]
    run_append(dtype, dim, page, "half", dim, new=[new] * seqs, start=start, ragged=False, seed=seqs, panel=seqs != 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (24, 3)])
def test_append_head_counts(dtype, heads, kv_heads):
    run_append(dtype, 128, 32, "interleaved", 128, new=[5, 60], start=[30, 1], heads=heads, kv_heads=kv_heads, seed=heads)


def test_append_many_ragged_sequences():
    new = [(b * 7) % 4 for b in range(1100)]
    run_append(FP8, 64, 16, "half", 64, new=new, start=[(b * 5) % 40 for b in range(1100)], heads=2, kv_heads=1)


def test_append_values_at_the_ends_of_the_formats():
    """Infinities saturate, NaN stays, zeros and tiny rows take the smallest scale, and none of them disturbs its neighbours."""
    from thor_megakernels_b200 import paged

    gen = generator(3)
    k, v, ks, vs = pool(FP8, 4, 1, 16, 64, gen)
    rows = torch.zeros((16, 1, 64), device="cuda")
    rows[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    rows[1, 0, 0] = 7.0          # 1.75 * 2^2: exactly the largest value of its scale
    bf = rows.bfloat16()
    table = ints([[2]])
    paged.append(bf, bf, k, v, table, ints([0]), k_scales=ks, v_scales=vs)
    for codes, scales in ((k, ks), (v, vs)):
        assert float(scales[2, 0]) == 2.0 ** -6
        x = codes[2, 0].float()
        assert x[0, 0] == 448 and x[0, 1] == -448 and torch.isnan(x[0, 2]) and x[0, 3] * 2.0 ** -6 == 3.0 and x[1, 0] == 448
        assert (x[2:] == 0).all()
    paged.append(torch.zeros_like(bf), torch.full_like(bf, 1e-30), k, v, table, ints([0]), k_scales=ks, v_scales=vs)
    assert float(ks[2, 0]) == 2.0 ** -64 and float(vs[2, 0]) == 2.0 ** -64 and (k[2].float() == 0).all()
    big = torch.full((1, 1, 64), 3.0e38, device="cuda").bfloat16()
    paged.append(big, big, k, v, table, ints([15]), k_scales=ks, v_scales=vs)
    assert float(ks[2, 0]) == 2.0 ** 120
    assert abs(float(k[2, 0, 15, 0].float()) * 2.0 ** 120 / float(big[0, 0, 0]) - 1) <= 2.0 ** -4
    assert (v[2, 0, :15].float() == 0).all()
    paged.check_errors()


def test_append_one_by_one_equals_the_rule():
    """Rows of growing magnitude arrive singly: the scale follows the largest so far, earlier codes follow the scale."""
    from thor_megakernels_b200 import paged

    gen = generator(4)
    k, v, ks, vs = pool(FP8, 3, 2, 32, 128, gen, spread=4.0)
    rows = torch.randn((40, 2, 128), generator=gen, device="cuda") * torch.exp2(torch.arange(40, device="cuda") / 3)[:, None, None]
    rows = rows.bfloat16()
    table = ints([[1, 2]])
    for i in range(40):
        paged.append(rows[i:i + 1], rows[i:i + 1], k, v, table, ints([i]), k_scales=ks, v_scales=vs)
    for page, lo, hi in ((1, 0, 32), (2, 32, 40)):
        for h in range(2):
            want = rows[lo:hi, h].double()
            sc = po.scale_for(float(want.abs().max()))
            assert float(ks[page, h]) == sc == float(vs[page, h])
            # rounded once, and again only where a code became subnormal: each step below half a subnormal
            assert ((k[page, h, :hi - lo].double() * sc - want).abs() <= 2.0 ** -4 * want.abs() + 2 * sc * 2.0 ** -10).all()
    paged.check_errors()


def test_append_bad_pages_and_positions_are_left_out_and_reported():
    from thor_megakernels_b200 import paged
    from thor_megakernels_b200._lib import MegakernelError

    gen = generator(5)
    for dtype in DTYPES:
        k, v, ks, vs = pool(dtype, 4, 1, 16, 64, gen)
        before = [t.clone() for t in (k, v)]
        rows = torch.randn((3, 1, 64), generator=gen, device="cuda").bfloat16()
        scales = dict(k_scales=ks, v_scales=vs)
        paged.append(rows, rows, k, v, ints([[-1], [-7], [-1]]), ints([0, 1, 2]), **scales)   # no page: nothing kept, no error
        paged.check_errors()
        paged.append(rows, rows, k, v, ints([[4], [2 ** 30], [-1]]), ints([0, 1, 2]), **scales)
        with pytest.raises(MegakernelError):
            paged.check_errors()
        paged.append(rows, rows, k, v, ints([[0], [1], [2]]), ints([16, 2 ** 31 - 1, 17]), **scales)
        with pytest.raises(MegakernelError):
            paged.check_errors()
        paged.check_errors()   # reported once
        for a, b in zip((k, v), before):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# --------------------------------------------------------------------------- attention

def run_attention(dtype, dim, page, heads, kv_heads, new, lengths, ragged=True, seed=0, scale=None, spread=1.0, q_size=2.0):
    from thor_megakernels_b200 import paged

    gen = generator(seed)
    pages = sum(-(-n // page) for n in lengths) + 2
    k, v, ks, vs = pool(dtype, pages, kv_heads, page, dim, gen, spread)
    table = page_table([max(1, n) for n in lengths], page, pages, gen, extra_columns=1)
    tokens = sum(new)
    cu = ints([0] + list(torch.tensor(new).cumsum(0))) if ragged else None
    q = (torch.randn((tokens, heads, dim), generator=gen, device="cuda") * q_size).bfloat16()
    scale = 1 / math.sqrt(dim) if scale is None else scale
    got = paged.attention(q, k, v, table, ints(lengths), scale=scale, k_scales=ks, v_scales=vs, cu_tokens=cu)
    paged.check_errors()
    check_attention(got, q, k, v, ks, vs, table, ints(lengths), cu, page, scale)
    again = paged.attention(q, k, v, table, ints(lengths), scale=scale, k_scales=ks, v_scales=vs, cu_tokens=cu)
    assert torch.equal(got, again)   # no atomics: the same bits


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 64), (128, 16), (128, 32), (128, 128)])
def test_decode_lengths(dtype, dim, page):
    lengths = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 511, 1025]
    run_attention(dtype, dim, page, 8, 2, [1] * len(lengths), lengths, ragged=False, seed=page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,new", [(1, 1, 1), (7, 1, 1), (8, 1, 1), (12, 1, 2), (16, 1, 1), (6, 2, 3), (8, 8, 9), (20, 4, 5), (32, 1, 2)])
def test_groups_and_drafted_tokens(dtype, heads, kv_heads, new):
    lengths = [new, new + 1, 64, 65 + new, 130, max(0, new - 1), 700]
    run_attention(dtype, 64 if heads % 3 else 128, 32, heads, kv_heads, [new] * len(lengths), lengths, ragged=False, seed=heads + new)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page", [(64, 64), (128, 16), (128, 64)])
def test_ragged_prompts(dtype, dim, page):
    run_attention(dtype, dim, page, 4, 1, new=[70, 1, 0, 33, 5, 128], lengths=[70, 300, 9, 40, 5, 400], seed=dim)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_long_sequence_is_split(dtype):
    run_attention(dtype, 128, 64, 4, 1, [1, 1], [9001, 12], ragged=False, seed=9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_peaked_scores_and_uneven_pages(dtype):
    """Scores of some hundreds, pages whose magnitudes differ by factors of thousands."""
    run_attention(dtype, 64, 16, 4, 1, [2, 1], [500, 200], seed=1, scale=1.0, spread=5.0, q_size=4.0)


def test_e4m3_pages_of_zeros_and_of_tiny_values():
    from thor_megakernels_b200 import paged

    gen = generator(12)
    k, v, ks, vs = pool(FP8, 6, 1, 16, 64, gen)
    vs[1], ks[1] = 2.0 ** -64, 2.0 ** -64
    vs[3] = 0.0
    table, lengths = ints([[1, 0, 3, 2, 4, 5]]), ints([90])
    q = torch.randn((1, 4, 64), generator=gen, device="cuda").bfloat16()
    got = paged.attention(q, k, v, table, lengths, k_scales=ks, v_scales=vs)
    check_attention(got, q, k, v, ks, vs, table, lengths, None, 16, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
def test_query_rows_of_any_size(dtype):
    from thor_megakernels_b200 import paged

    gen = generator(13)
    k, v, ks, vs = pool(dtype, 4, 1, 32, 64, gen)
    q = torch.randn((4, 4, 64), generator=gen, device="cuda")
    q = (q * torch.tensor([1e-20, 1e-4, 0.0, 200.0], device="cuda")[:, None, None]).bfloat16()
    table, lengths = ints([[0], [1], [2], [3]]), ints([32, 20, 7, 32])
    scale = 0.05
    got = paged.attention(q, k, v, table, lengths, scale=scale, k_scales=ks, v_scales=vs)
    check_attention(got, q, k, v, ks, vs, table, lengths, None, 32, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 5, 40])
def test_what_is_not_finite_stays_where_it_is_seen(dtype, new):
    """NaN behind the last position, in unused pages and in tokens of the future reaches nobody who does not see it."""
    from thor_megakernels_b200 import paged

    gen = generator(14)
    k, v, ks, vs = pool(dtype, 8, 1, 32, 64, gen)
    length = 100
    table, lengths = ints([[6, 1, 4, 3]]), ints([length])
    clean_k, clean_v = k.clone(), v.clone()
    nan = torch.full((64,), math.nan, device="cuda").to(dtype)
    for t in (k, v):
        t[3, 0, length - 96:] = nan     # behind the end
        t[[0, 2, 5, 7]] = nan           # pages of nobody
    q = torch.randn((new, 4, 64), generator=gen, device="cuda").bfloat16()
    cu = ints([0, new])
    args = dict(k_scales=ks, v_scales=vs, cu_tokens=cu)
    got = paged.attention(q, k, v, table, lengths, **args)
    want = paged.attention(q, clean_k, clean_v, table, lengths, **args)
    assert torch.equal(got, want)
    if new > 1:   # the last but one token's value and key are NaN: the rows before it do not know
        v[3, 0, length - 96 - 2, 5] = nan[0]
        got = paged.attention(q, k, v, table, lengths, **args)
        assert torch.equal(got[:-2], want[:-2])
        assert torch.isnan(got[-2:, :, 5]).all()
        keep = torch.arange(64, device="cuda") != 5
        assert torch.equal(got[-2:][..., keep], want[-2:][..., keep])
        k[3, 0, length - 96 - 2, 5] = nan[0]
        got = paged.attention(q, k, v, table, lengths, **args)
        assert torch.equal(got[:-2], want[:-2]) and torch.isnan(got[-2:]).all()
    paged.check_errors()


def test_missing_and_bad_pages_take_no_part():
    from thor_megakernels_b200 import paged
    from thor_megakernels_b200._lib import MegakernelError

    gen = generator(15)
    for dtype in DTYPES:
        k, v, ks, vs = pool(dtype, 8, 2, 16, 64, gen)
        q = torch.randn((2, 4, 64), generator=gen, device="cuda").bfloat16()
        table, lengths = ints([[-1, 3, -1, 5], [-1, -1, -1, -1]]), ints([60, 40])
        got = paged.attention(q, k, v, table, lengths, k_scales=ks, v_scales=vs)
        paged.check_errors()
        check_attention(got, q, k, v, ks, vs, table, lengths, None, 16, 0.125)
        assert (got[1] == 0).all()
        table[0, 1] = 8
        got = paged.attention(q, k, v, table, lengths, k_scales=ks, v_scales=vs)
        with pytest.raises(MegakernelError):
            paged.check_errors()
        check_attention(got, q, k, v, ks, vs, table, lengths, None, 16, 0.125)
        got = paged.attention(q, k, v, ints([[1], [2]]), ints([17, -3]), k_scales=ks, v_scales=vs)   # longer than the table; negative
        with pytest.raises(MegakernelError):
            paged.check_errors()
        check_attention(got, q, k, v, ks, vs, ints([[1], [2]]), ints([16, 0]), None, 16, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_layouts(dtype):
    """A dense cache [batch, positions, heads, dim] seen as pages, queries inside a wider panel, a page table inside a wider one."""
    from thor_megakernels_b200 import paged

    gen = generator(16)
    k, v, ks, vs = pool(dtype, 3 * 8, 2, 32, 128, gen)
    dense = [t.transpose(1, 2).contiguous().view(3, 256, 2, 128) for t in (k, v)]
    seen = [t.view(24, 32, 2, 128).transpose(1, 2) for t in dense]
    wide = torch.full((3, 20), 99, dtype=torch.int32, device="cuda")
    wide[:, :8] = torch.arange(24, device="cuda").view(3, 8)
    table = wide[:, :8]
    panel = torch.randn((3, 12, 128), generator=gen, device="cuda").bfloat16()
    q, lengths = panel[:, 2:10], ints([256, 33, 100])
    got = paged.attention(q, *seen, table, lengths, k_scales=ks, v_scales=vs)
    paged.check_errors()
    check_attention(got, q, k, v, ks, vs, table, lengths, None, 32, 1 / math.sqrt(128))


def test_append_through_a_dense_view():
    from thor_megakernels_b200 import paged

    gen = generator(17)
    dense = [torch.randn((2, 64, 2, 64), generator=gen, device="cuda").bfloat16() for _ in range(2)]
    before = [t.clone() for t in dense]
    k, v = (t.view(4, 32, 2, 64).transpose(1, 2) for t in dense)
    rows = [torch.randn((2, 2, 64), generator=gen, device="cuda").bfloat16() for _ in range(2)]
    paged.append(*rows, k, v, ints([[0, 1], [2, 3]]), ints([5, 40]))
    for t, b, r in zip(dense, before, rows):
        b[0, 5], b[1, 40] = r[0], r[1]
        assert torch.equal(t, b)


def test_rows_of_no_sequence_stay_as_they_were():
    from thor_megakernels_b200 import paged

    gen = generator(18)
    k, v, _, _ = pool(torch.bfloat16, 4, 1, 16, 64, gen)
    q = torch.randn((9, 2, 64), generator=gen, device="cuda").bfloat16()
    out = torch.full_like(q, 5.0)
    paged.attention(q, k, v, ints([[0, 1], [2, 3]]), ints([20, 4]), cu_tokens=ints([1, 3, 7]), out=out)
    assert (out[0] == 5).all() and (out[7:] == 5).all() and (out[1:7] != 5).any(dim=2).all()
    kept = [t.clone() for t in (k, v)]
    q_out = torch.full_like(q, 5.0)
    paged.append(q[:, :1], q[:, 1:], k, v, ints([[0, 1], [2, 3]]), ints([20, 4]), q=q, q_out=q_out, cu_tokens=ints([1, 3, 7]))
    assert (q_out[0] == 5).all() and (q_out[7:] == 5).all() and torch.equal(q_out[1:7], q[1:7])
    for t, b, head in ((k, kept[0], 0), (v, kept[1], 1)):
        b[1, 0, 4:6], b[2, 0, 4:8] = q[1:3, head], q[3:7, head]
        assert torch.equal(t, b)
    paged.check_errors()


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB: pages at its end are where they should be."""
    from thor_megakernels_b200 import paged

    gen = generator(19)
    pages = 34000   # x 8 heads x 128 slots x 128 bytes = 4.5 GB of keys
    k, v = (torch.empty((pages, 8, 128, 128), dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
    ks, vs = (torch.ones((pages, 8), device="cuda") for _ in range(2))
    table = ints([[pages - 1, pages - 2, 0]])
    rows = [torch.randn((300, 8, 128), generator=gen, device="cuda").bfloat16() for _ in range(2)]
    paged.append(*rows, k, v, table, ints([0]), k_scales=ks, v_scales=vs)
    q = torch.randn((1, 8, 128), generator=gen, device="cuda").bfloat16()
    got = paged.attention(q, k, v, table, ints([300]), k_scales=ks, v_scales=vs)
    paged.check_errors()
    at = [pages - 1, pages - 2, 0]
    small = [torch.stack([t[i] for i in at]) for t in (k, v, ks, vs)]
    for codes, scales, r in ((small[0], small[2], rows[0]), (small[1], small[3], rows[1])):
        back = po.dequantise(codes, scales).transpose(1, 2).reshape(384, 8, 128)[:300]
        assert ((back - r.double()).abs() <= 2.0 ** -4 * r.double().abs() + float(scales.max()) * 2.0 ** -10).all()
    check_attention(got, q, *small, ints([[0, 1, 2]]), ints([300]), None, 128, 1 / math.sqrt(128))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page,heads,kv_heads,new,lengths", [
    (128, 64, 4, 1, [256], [256]),                                  # whole tiles, one row block pair
    (128, 128, 1, 1, [300], [1000]),                                # no groups
    (64, 16, 8, 1, [33], [33]),                                     # one row more than two whole tiles
    (64, 32, 28, 4, [70, 65, 9], [70, 400, 700]),                   # groups of 7: blocks end inside a token
    (128, 16, 16, 8, [200, 1, 17, 130], [457, 513, 17, 129]),       # fewer positions than rows; few-row sequences between
    (128, 32, 8, 2, [64] * 40, [64 + 3 * b for b in range(40)]),    # a CTA per row block
    (64, 64, 4, 1, [129, 0, 400], [129, 0, 2500]),
])
def test_prompts(dtype, dim, page, heads, kv_heads, new, lengths):
    run_attention(dtype, dim, page, heads, kv_heads, new, lengths, seed=dim + page + heads)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_with_a_negative_scale_and_peaked_scores(dtype):
    run_attention(dtype, 64, 16, 4, 1, [100, 40], [150, 300], seed=31, scale=-0.7, spread=3.0, q_size=3.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_over_missing_pages_and_idle_sequences(dtype):
    from thor_megakernels_b200 import paged

    gen = generator(32)
    k, v, ks, vs = pool(dtype, 40, 2, 16, 128, gen)
    q = torch.randn((150, 8, 128), generator=gen, device="cuda").bfloat16()
    table = torch.randperm(40, generator=gen, device="cuda").int()[:36].view(3, 12).contiguous()
    table[0, 0:8], table[0, 10], table[1] = -1, -1, -1
    table = torch.cat((table, table.new_full((3, 1), -1)), dim=1)
    lengths, cu = ints([190, 100, 0]), ints([0, 60, 110, 150])
    got = paged.attention(q, k, v, table, lengths, k_scales=ks, v_scales=vs, cu_tokens=cu)
    paged.check_errors()
    check_attention(got, q, k, v, ks, vs, table, lengths, cu, 16, 1 / math.sqrt(128))
    assert (got[60:] == 0).all()


# --------------------------------------------------------------------------- use

@pytest.mark.parametrize("dtype", DTYPES)
def test_decoding_step_by_step_equals_the_prompt_at_once(dtype):
    """Append and attention token by token, in chunks, and all at once see the same cache; a captured step replays."""
    from thor_megakernels_b200 import paged

    gen = generator(20)
    n, heads, kv_heads, dim, page = 45, 4, 2, 64, 16
    x = torch.randn((n, heads + 2 * kv_heads, dim), generator=gen, device="cuda").bfloat16()
    q, kn, vn = x.split((heads, kv_heads, kv_heads), dim=1)
    angle = torch.rand((64, dim), generator=gen, device="cuda")
    rope = dict(rope_cos=angle.cos(), rope_sin=angle.sin(), layout="half")
    table = ints([[2, 0, 3]])

    def fresh():
        k, v, ks, vs = pool(dtype, 4, kv_heads, page, dim, generator(1))
        return (k, v), dict(k_scales=ks, v_scales=vs)

    def step(cache, scales, lo, hi, start, lengths):
        r = paged.append(kn[lo:hi], vn[lo:hi], *cache, table, start, q=q[lo:hi], **rope, **scales)
        return paged.attention(r, *cache, table, lengths, **scales)

    cache, scales = fresh()
    whole = step(cache, scales, 0, n, ints([0]), ints([n]))
    cache2, scales2 = fresh()
    chunks = torch.cat([step(cache2, scales2, lo, min(lo + 16, n), ints([lo]), ints([min(lo + 16, n)])) for lo in range(0, n, 16)])
    # pages end where chunks do, so the scales are those of the whole prompt and the codes are the same
    for a, b in zip(cache, cache2):
        for i, p in enumerate((2, 0, 3)):
            used = min(page, n - i * page)
            assert torch.equal(a[p, :, :used].view(torch.uint8), b[p, :, :used].view(torch.uint8))
    # Two roundings of the result (2^-8 each) and the two calls' weights: the prompt at once has 90 rows per KV head and so one bf16
    # term per weight (2^-8 of sum w |v| <= max |v|), chunks of at most 32 rows have two (2^-16); f16 weights (2^-11) for E4M3.
    mag = vn.abs().double().max()
    apart = 2.0 ** -7 * whole.double().abs() + ((2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -10) + 2.0 ** -13) * mag
    assert ((whole.double() - chunks.double()).abs() <= apart).all()
    if dtype == torch.bfloat16:   # 8-bit: earlier rows were read with an earlier scale of their page
        cache3, scales3 = fresh()
        single = torch.cat([step(cache3, scales3, i, i + 1, ints([i]), ints([i + 1])) for i in range(n)])
        assert ((whole.double() - single.double()).abs() <= apart).all()
        assert ((chunks.double() - single.double()).abs() <= 2.0 ** -7 * whole.double().abs() + 2.0 ** -13 * mag).all()

    # one decode step captured, replayed over positions that device data names
    cache4, scales4 = fresh()
    step(cache4, scales4, 0, 32, ints([0]), ints([32]))
    start, lengths = ints([32]), ints([33])
    row = [t[32:33].clone() for t in (q, kn, vn)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = paged.append(row[1], row[2], *cache4, table, start, q=row[0], **rope, **scales4)
        paged.attention(warm, *cache4, table, lengths, **scales4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = paged.append(row[1], row[2], *cache4, table, start, q=row[0], **rope, **scales4)
        out = paged.attention(r, *cache4, table, lengths, **scales4)
    cache5, scales5 = fresh()
    step(cache5, scales5, 0, 32, ints([0]), ints([32]))
    for i in range(32, n):
        for dst, src in zip(row, (q, kn, vn)):
            dst.copy_(src[i:i + 1])
        start.fill_(i)
        lengths.fill_(i + 1)
        graph.replay()
        want = step(cache5, scales5, i, i + 1, ints([i]), ints([i + 1]))
        assert torch.equal(out, want)
    paged.check_errors()


def test_calls_on_two_streams_do_not_disturb_one_another():
    from thor_megakernels_b200 import paged

    gen = generator(21)
    sets = []
    for i in range(2):
        k, v, ks, vs = pool(FP8, 200, 2, 64, 128, gen)
        q = torch.randn((3, 8, 128), generator=gen, device="cuda").bfloat16()
        table = torch.randperm(200, generator=gen, device="cuda").int()[:195].view(3, 65).contiguous()
        sets.append((q, k, v, table, ints([4100, 2000, 77]), dict(k_scales=ks, v_scales=vs)))
    want = [paged.attention(*s[:5], **s[5]) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(paged.attention(*sets[i][:5], **sets[i][5]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_own_workspace():
    from thor_megakernels_b200 import _lib, paged

    gen = generator(22)
    k, v, _, _ = pool(torch.bfloat16, 40, 1, 64, 64, gen)
    q = torch.randn((1, 4, 64), generator=gen, device="cuda").bfloat16()
    table, lengths = torch.arange(40, device="cuda").int().view(1, 40), ints([2500])
    need = paged.attention_workspace(q, k, v, table, lengths)
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")   # contents do not matter
    assert torch.equal(paged.attention(q, k, v, table, lengths, workspace=ws), paged.attention(q, k, v, table, lengths))
    with pytest.raises(_lib.MegakernelError):
        paged.attention(q, k, v, table, lengths, workspace=ws[: need - 16])


def test_refusals_on_the_device():
    from thor_megakernels_b200 import paged
    from thor_megakernels_b200._lib import MegakernelError

    gen = generator(23)
    k, v, _, _ = pool(torch.bfloat16, 4, 2, 16, 64, gen)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device="cuda")
    table, one = ints([[0, 1]]), ints([1])
    ok = (q, k, v, table, one)
    paged.attention(*ok)

    def refused(call, *args, kinds=(ValueError, MegakernelError), **kw):
        with pytest.raises(kinds):
            call(*args, **kw)

    refused(paged.attention, q[:, :3], k, v, table, one)                       # 3 query heads over 2
    refused(paged.attention, q.half(), k, v, table, one)
    refused(paged.attention, q, k.half(), v.half(), table, one)
    refused(paged.attention, q, k, v[:2], table, one)
    refused(paged.attention, q, k, v, table.long(), one)
    refused(paged.attention, q, k, v, table, one.float())
    refused(paged.attention, q, k, v, table, ints([1, 2]))
    refused(paged.attention, q, k, v, table, one.cpu())
    refused(paged.attention, q, k, v, table, one, cu_tokens=ints([0, 1, 1]))
    refused(paged.attention, q, k, v, table, one, k_scales=torch.ones((4, 2), device="cuda"))
    refused(paged.attention, q, k.to(FP8), v.to(FP8), table, one)              # no scales
    refused(paged.attention, q, k[..., :32], v[..., :32], table, one)
    refused(paged.attention, q[..., :32], k[..., :32].contiguous(), v[..., :32].contiguous(), table, one)
    refused(paged.attention, q, k[:, :, :12], v[:, :, :12], table, one)        # page size 12
    refused(paged.attention, q, k, v, table, one, out=torch.zeros((1, 4, 32), dtype=torch.bfloat16, device="cuda"))
    refused(paged.attention, q, k, v, table, one, scale=math.nan)
    refused(paged.attention, torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda"), k, v, ints([[0], [1]]), ints([1, 1]))
    rows = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    cos = torch.ones((8, 64), device="cuda")
    refused(paged.append, rows, rows[:, :1], k, v, table, one)
    refused(paged.append, rows, rows, k, v, table, one, rope_cos=cos)
    refused(paged.append, rows, rows, k, v, table, one, rope_cos=cos[:, :24].contiguous(), rope_sin=cos[:, :24].contiguous())
    refused(paged.append, rows, rows, k, v, table, one, rope_cos=cos.double(), rope_sin=cos.double())
    refused(paged.append, rows, rows, k, v, table, one, layout="neox")
    refused(paged.append, rows, rows, k, v, table, one, q_out=q)
    refused(paged.append, rows, rows, k, v, table, one, q=q[..., 1:])
    odd = torch.zeros(2 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(1, 2, 64)
    refused(paged.append, odd, rows, k, v, table, one)                         # not on a 16-byte boundary
    assert paged.attention(q[:0], k, v, table[:0], one[:0], cu_tokens=ints([0])).shape == (0, 4, 64)
    paged.check_errors()


# --------------------------------------------------------------------------- calls that are easy to forget

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 3], [70, 9]])
@pytest.mark.parametrize("scale", [-0.7, 0.0])
def test_negative_and_zero_scales(dtype, new, scale):
    run_attention(dtype, 64, 16, 4, 1, new, [150, 300], seed=41, scale=scale, q_size=3.0)


@pytest.mark.parametrize("layout,rot", [("interleaved", 64), ("half", 32)])
def test_rotation_in_place(layout, rot):
    from thor_megakernels_b200 import paged

    gen = generator(42)
    k, v, _, _ = pool(torch.bfloat16, 8, 2, 16, 64, gen)
    rows = torch.randn((37, 2, 64), generator=gen, device="cuda").bfloat16()
    q = torch.randn((37, 9, 64), generator=gen, device="cuda").bfloat16()
    angle = torch.rand((64, rot), generator=gen, device="cuda") * 6
    args = (rows, rows, k, v, torch.arange(3, device="cuda").int().view(1, 3), ints([5]))
    tables = dict(rope_cos=angle.cos(), rope_sin=angle.sin(), layout=layout)
    want = paged.append(*args, q=q, **tables)
    got = paged.append(*args, q=q, q_out=q, **tables)
    assert got is q and torch.equal(got, want)
    paged.check_errors()


def test_overlapping_outputs_are_refused():
    from thor_megakernels_b200 import paged

    k, v, _, _ = pool(torch.bfloat16, 4, 2, 16, 64, generator(43))
    buffer = torch.zeros((6, 4, 64), dtype=torch.bfloat16, device="cuda")
    q, table, start = buffer[:4], ints([[0, 1]]), ints([0])
    rows = buffer.view(12, 2, 64)[:4]
    other = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        paged.attention(q, k, v, table, ints([4]), out=q)
    with pytest.raises(ValueError, match="overlap"):
        paged.attention(q, k, v, table, ints([4]), out=buffer[2:])
    with pytest.raises(ValueError, match="overlap"):
        paged.append(other, other, k, v, table, start, q=q, q_out=buffer[2:])
    with pytest.raises(ValueError, match="overlap"):
        paged.append(rows, other, k, v, table, start, q=torch.zeros_like(q), q_out=q)
    packed = torch.zeros((1, 8, 64), dtype=torch.bfloat16, device="cuda")   # side by side is not overlapping
    paged.append(packed[:, 4:6], packed[:, 6:], k, v, table, start, q=packed[:, :4], q_out=packed[:, :4])
    paged.check_errors()


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_that_do_not_grow_are_reported(dtype):
    """Rows and pages of no sequence stay as they were, and the next call is right."""
    from thor_megakernels_b200 import paged
    from thor_megakernels_b200._lib import MegakernelError

    gen = generator(44)
    k, v, ks, vs = pool(dtype, 40, 2, 16, 64, gen)
    rows = torch.randn((64, 2, 64), generator=gen, device="cuda").bfloat16()
    q = torch.randn((64, 8, 64), generator=gen, device="cuda").bfloat16()
    table = torch.arange(30, device="cuda").int().view(5, 6)
    scales = dict(k_scales=ks, v_scales=vs)
    for cu in ([0, 50, 20, 64, 3, 64], [60, 40, 20, 10, 5, 0], [-5, 70, 2 ** 31 - 1, -2 ** 31, 8, 64], [64, 0, 64, 0, 64, 0]):
        kept = [t[30:].clone() for t in (k, v)]
        paged.append(rows, rows, k, v, table, ints([3, 0, 17, 20, 1]), q=q, cu_tokens=ints(cu), **scales)
        with pytest.raises(MegakernelError):
            paged.check_errors()
        for a, b in zip((k, v), kept):
            assert torch.equal(a[30:].view(torch.uint8), b.view(torch.uint8))
        out = paged.attention(q, k, v, table, ints([80, 96, 60, 90, 70]), cu_tokens=ints(cu), **scales)
        assert out.shape == q.shape
        with pytest.raises(MegakernelError):
            paged.check_errors()
    run_attention(dtype, 64, 16, 8, 2, [40, 24], [80, 96], seed=45)


def test_offsets_that_repeat_all_rows_for_many_sequences():
    """512 sequences claim the same 4096 rows over a million positions each: more work than an int counts.  Nothing is done.
    (256 row blocks x 4 KV heads x at least 8160 tiles x 512 = 4.3e9; with a group of 8 heads it would be 2.144e9, just below.)"""
    from thor_megakernels_b200 import paged
    from thor_megakernels_b200._lib import MegakernelError

    k, v, _, _ = pool(torch.bfloat16, 2, 4, 128, 64, generator(46))
    q = torch.ones((4096, 64, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.full((1024, 8192), -1, dtype=torch.int32, device="cuda")
    lengths = torch.full((1024,), 1 << 20, dtype=torch.int32, device="cuda")
    cu = ints([0, 4096] * 512 + [0])
    out = torch.full_like(q, 7.0)
    paged.attention(q, k, v, table, lengths, cu_tokens=cu, out=out)
    with pytest.raises(MegakernelError):
        paged.check_errors()
    assert (out == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_append_and_attention_follow_their_inputs(dtype):
    from thor_megakernels_b200 import paged

    gen = generator(47)
    pools = [pool(dtype, 40, 2, 32, 64, generator(48)) for _ in range(2)]   # alike
    table = torch.randperm(40, generator=gen, device="cuda").int().view(4, 10)
    steps = [(ints(s), [torch.randn((4 * n, h, 64), generator=gen, device="cuda").bfloat16() for h in (8, 2, 2)])
             for n, s in ((3, [0, 5, 100, 250]), (3, [3, 8, 103, 253]), (3, [6, 11, -1, 256]))]
    angle = torch.rand((320, 64), generator=gen, device="cuda") * 6
    cos, sin = angle.cos(), angle.sin()

    def step(p, start, q, k, v):
        scales = dict(k_scales=p[2], v_scales=p[3])
        rotated = paged.append(k, v, p[0], p[1], table, start, q=q, rope_cos=cos, rope_sin=sin, q_out=torch.zeros_like(q), **scales)
        return paged.attention(rotated, p[0], p[1], table, torch.where(start < 0, 0, start + 3).int(), **scales)

    want = [step(pools[0], start, *rows) for start, rows in steps]
    start, rows = steps[0][0].clone(), [t.clone() for t in steps[0][1]]
    start.fill_(-1)
    step(pools[1], start, *rows)   # idle: stores nothing
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(pools[1], start, *rows)
    for (s, r), w in zip(steps, want):
        start.copy_(s)
        for a, b in zip(rows, r):
            a.copy_(b)
        graph.replay()
        assert torch.equal(got, w)
    paged.check_errors()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_cache_layer_by_layer(dtype):
    """A prompt, then single tokens of two of three sequences, through PagedKvCache.layer."""
    from thor_megakernels_b200 import paged

    gen = generator(49)
    cache = paged.PagedKvCache(2, 20, 2, 64, page_size=16, max_seqs=3, max_positions=96, dtype=dtype)
    lengths = [37, 16]
    for b, n in enumerate(lengths):
        cache.reserve(b, n + 2)
    cu, start = ints([0, 37, 53]), ints([0, 0])
    for new, at, offsets in ((53, start, cu), (2, ints(lengths), None), (2, ints([n + 1 for n in lengths]), None)):
        seen = at + (ints(lengths) if offsets is not None else 1)
        for layer in range(2):
            k, v = (torch.randn((new, 2, 64), generator=gen, device="cuda").bfloat16() for _ in range(2))
            q = torch.randn((new, 6, 64), generator=gen, device="cuda").bfloat16()
            args = cache.layer(layer, 2)
            paged.append(k, v, **args, start=at, cu_tokens=offsets)
            got = paged.attention(q, **args, lengths=seen, cu_tokens=offsets)
            paged.check_errors()
            check_attention(got, q, args["k_pages"], args["v_pages"], args.get("k_scales"), args.get("v_scales"), args["page_table"], seen, offsets, 16, 1 / 8)
    for b in range(2):
        cache.release(b)
    assert cache.free_pages == 20


@pytest.mark.parametrize("new", [1, 40])
def test_value_scales_far_apart_and_zero(new):
    """Equal scores over pages whose values are 2^90 apart: the denominator counts both; a scale of 0 makes a page of zeros."""
    from thor_megakernels_b200 import paged

    gen = generator(50)
    k = torch.zeros((4, 1, 64, 64), device="cuda").to(FP8)
    v = torch.randint(1, 5, (4, 1, 64, 64), generator=gen, device="cuda").float().to(FP8)
    ks = torch.ones((4, 1), device="cuda")
    q = torch.randn((new, 4, 64), generator=gen, device="cuda").bfloat16()
    table, lengths = ints([[1, 3, 0]]), ints([192])
    for scales in ([2.0 ** 60, 1.0, 9.0, 2.0 ** -30], [2.0, 1.0, 9.0, 0.0]):
        vs = torch.tensor(scales, device="cuda").view(4, 1)
        got = paged.attention(q, k, v, table, lengths, k_scales=ks, v_scales=vs)
        paged.check_errors()
        check_attention(got, q, k, v, ks, vs, table, lengths, None, 64, 1 / 8)
