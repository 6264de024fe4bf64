"""BatchedDecoder over a paged cache: the same model, tokens and positions as over the dense cache."""
import pytest
import torch

from helpers import assert_close, nrmse

pytestmark = pytest.mark.gpu

CFG = dict(hidden_size=2048, num_hidden_layers=2, num_attention_heads=32, num_key_value_heads=8, head_dim=64, intermediate_size=8192,
           vocab_size=4096)


def build(cfg=CFG, batch=8, max_len=512):
    from thor_megakernels_b200.llama import LlamaConfig, LlamaForCausalLM
    from thor_megakernels_b200.model_types import ExtraModelConfig

    return LlamaForCausalLM.random_init(LlamaConfig(**cfg), ExtraModelConfig(interleave_rope=True, max_len_override=max_len, max_batch_size=batch),
                                        seed=3, device="cuda")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def run(model, cache, prompts, steps):
    """Prefill the prompts into their slots, then decode greedily with the tokens of ``steps``; all logits."""
    from thor_megakernels_b200.batched import BatchedDecoder

    dec = BatchedDecoder(model, 128 if cache is None else 100, cache=cache)
    logits, lengths = [], []
    for slot, prompt in enumerate(prompts):
        if cache is not None:
            cache.reserve(slot, len(prompt))
        dec.prefill(ints(prompt), slot=slot)
        logits.append(dec.logits[:1].float().clone())
        lengths.append(len(prompt))
    for tokens in steps:
        if cache is not None:
            for b, n in enumerate(lengths):
                cache.reserve(b, n + 1)
        dec.step(ints(tokens), ints(lengths))
        logits.append(dec.logits[: len(tokens)].float().clone())
        lengths = [n + 1 for n in lengths]
    dec.status()
    dec.close()
    return logits


def inputs(seed=5):
    gen = torch.Generator().manual_seed(seed)
    prompts = [torch.randint(0, 4096, (n,), generator=gen).tolist() for n in (1, 37, 128, 250, 64)]
    steps = [torch.randint(0, 4096, (5,), generator=gen).tolist() for _ in range(6)]
    return prompts, steps


@pytest.mark.parametrize("page_size", [16, 64])
def test_bf16_pages_equal_the_dense_cache(page_size):
    """The two caches hold the same rows; the attention kernels differ in the order of fp32 sums and (prompt passes of more than 32
    rows per KV head) in weights of one bf16 term, 2^-8 of the weighted values.  Two layers of single-ulp flips: the stated band,
    or relative 2-norm 2^-6 of the logits where it is left."""
    from thor_megakernels_b200.paged import PagedKvCache

    model = build()
    prompts, steps = inputs()
    cache = PagedKvCache.for_model(model, 80, page_size=page_size, max_seqs=6, max_positions=400)
    free = cache.free_pages
    want, got = run(model, None, prompts, steps), run(model, cache, prompts, steps)
    for a, b in zip(got, want):
        assert nrmse(a, b) <= 2.0 ** -6
    assert_close("first prompt of one token", got[0], want[0])
    for b in range(5):
        cache.release(b)
    assert cache.free_pages == free and (cache.page_table == -1).all()


def test_e4m3_pages_follow_the_dense_cache():
    """Keys and values lose at most 2^-4 of themselves each (E4M3), so the attention's part of the residual stream moves by no more
    than about 2^-3."""
    from thor_megakernels_b200.paged import PagedKvCache

    model = build()
    prompts, steps = inputs(6)
    cache = PagedKvCache.for_model(model, 40, page_size=32, max_seqs=5, dtype=torch.float8_e4m3fn)
    for a, b in zip(run(model, cache, prompts, steps), run(model, None, prompts, steps)):
        assert nrmse(a, b) <= 2.0 ** -3
    assert (cache.k_scales > 0).all()


def test_a_captured_step_follows_the_page_table():
    """One graph, replayed while sequences grow into new pages: the same logits as steps that are launched."""
    from thor_megakernels_b200.batched import BatchedDecoder
    from thor_megakernels_b200.paged import PagedKvCache

    model = build()
    prompts, steps = inputs(7)
    prompts, steps = prompts[:3], [s[:3] for s in steps]
    cache = PagedKvCache.for_model(model, 60, page_size=16, max_seqs=3)
    want = run(model, cache, prompts, steps)[3:]
    for b in range(3):
        cache.release(b)
    dec = BatchedDecoder(model, 8, cache=cache)
    for slot, prompt in enumerate(prompts):
        cache.reserve(slot, len(prompt))
        dec.prefill(ints(prompt), slot=slot)
    tokens, pos, out = ints(steps[0]), ints([len(p) for p in prompts]), torch.empty(3, dtype=torch.int32, device="cuda")
    start = pos.clone()
    for b, p in enumerate(prompts):
        cache.reserve(b, len(p) + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.step(tokens, pos, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dec.step(tokens, pos, out=out)
    for i, step in enumerate(steps):
        for b, p in enumerate(prompts):
            cache.reserve(b, len(p) + i + 1)
        tokens.copy_(ints(step))
        pos.copy_(start + i)
        graph.replay()
        # a prompt pass of other max_batch rows differs in its sums; steps are the same kernels on nearly the same rows
        assert nrmse(dec.logits[:3].float(), want[i]) <= 2.0 ** -6
        assert torch.equal(out.long(), dec.logits[:3].float().argmax(dim=1))
    dec.status()
    dec.close()


def test_rows_without_a_page_are_not_kept_and_bad_ids_are_reported():
    from thor_megakernels_b200._lib import MegakernelError
    from thor_megakernels_b200.batched import BatchedDecoder
    from thor_megakernels_b200.paged import PagedKvCache

    model = build(batch=2)
    cache = PagedKvCache.for_model(model, 4, page_size=16, max_seqs=4)
    dec = BatchedDecoder(model, 4, cache=cache)
    cache.reserve(1, 5)
    before = cache.k.clone()
    dec.step(ints([5, 6, 7]), ints([0, 20, 3]))   # sequences 0 and 2 have no page, sequence 1 none for position 20
    dec.status()
    assert torch.equal(cache.k.view(torch.int16), before.view(torch.int16))
    cache.page_table[0, 0] = 4
    dec.step(ints([5, 6, 7]), ints([0, 1, 3]))
    with pytest.raises(MegakernelError):
        dec.status()
    dec.status()
    with pytest.raises(ValueError):
        dec.step(ints([1, 2, 3, 4, 5]), ints([0, 0, 0, 0, 0]))
    with pytest.raises((ValueError, MegakernelError)):
        BatchedDecoder(model, 4, cache=PagedKvCache(2, 4, 4, 64, max_seqs=4))    # other heads
    with pytest.raises(ValueError):
        BatchedDecoder(model, 4, cache=PagedKvCache(3, 4, 8, 64, max_seqs=4))    # other layers
    dec.close()


def test_pages_are_handed_out_and_taken_back():
    from thor_megakernels_b200.paged import PagedKvCache

    cache = PagedKvCache(1, 5, 1, 64, page_size=16, max_seqs=3, max_positions=64)
    cache.reserve(0, 17)
    cache.reserve(0, 5)
    cache.reserve(1, 33)
    assert cache.free_pages == 0
    table = cache.page_table.tolist()
    assert sorted(i for row in table for i in row if i >= 0) == [0, 1, 2, 3, 4] and table[2] == [-1] * 4
    with pytest.raises(MemoryError):
        cache.reserve(2, 1)
    with pytest.raises(ValueError):
        cache.reserve(0, 65)
    cache.release(0)
    cache.reserve(2, 30)
    assert sorted(cache.page_table[2].tolist()) == sorted([-1, -1] + table[0][:2])
