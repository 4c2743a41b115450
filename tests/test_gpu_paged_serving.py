"""GPU tests of serving from the paged cache: steps that mix pieces of prompts and
single tokens against the batched plan and against themselves cut differently,
forks, and sampling end to end."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_decode import norm_close  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def setup():
    from kudacuda_b200.decode_engine import random_weights, tiny_config
    from kudacuda_b200.kudacuda_sidecar import KudaCudaBridge
    from kudacuda_b200.paged_serving import PagedGenerator

    torch.cuda.set_device(0)
    bridge = KudaCudaBridge(device_id=0)
    weights = random_weights(bridge, tiny_config(layers=2, vocab=4096), seed=17, device=DEV)
    gen = PagedGenerator(bridge, weights, num_pages=64, page_size=16, max_position=512, device=DEV)
    yield bridge, weights, gen
    bridge.shutdown()


def prompt(n, seed):
    return torch.randint(0, 4096, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def test_a_prompt_in_pieces_gives_what_single_tokens_give(setup):
    from kudacuda_b200.paged_serving import PagedSequence, Sampling

    _, _, gen = setup
    ids = prompt(90, 1)
    greedy = Sampling()
    finals = []
    for pieces in ([1] * 90, [64, 26], [7, 40, 1, 42]):
        seq, at = PagedSequence(), 0
        for n in pieces:
            gen.step([(seq, ids[at:at + n])], [greedy], [0.5])
            at += n
        finals.append((gen.x[pieces[-1] - 1].float().cpu().numpy(),
                       gen.cache.k[:, seq.pages[2], :, 3].float().cpu().numpy()))
        gen.cache.free(seq)
    for x, k in finals[1:]:
        norm_close(x, finals[0][0], 2e-2)  # 1e-2 a layer, as everywhere
        norm_close(k, finals[0][1], 2e-2)
    assert gen.cache.free_pages == 64


def test_paged_steps_agree_with_the_batched_plan(setup):
    """The same token at the same positions over the same prefix, contiguous and paged caches."""

    from kudacuda_b200.decode_engine import BatchedDecodePlan
    from kudacuda_b200.paged_serving import PagedSequence, Sampling

    bridge, weights, gen = setup
    lens = [1, 17, 40]
    prompts = [prompt(n, 10 + n) for n in lens]
    seqs = [PagedSequence() for _ in lens]
    gen.step([(s, p) for s, p in zip(seqs, prompts)], [Sampling()] * 3, [0.0] * 3)
    ours = [gen.x[sum(lens[:i + 1]) - 1].float().cpu().numpy() for i in range(3)]
    plan = BatchedDecodePlan(bridge, weights, batch=3, kv_bucket=64, max_tokens=64, device=DEV)
    stream = torch.cuda.Stream()
    plan.capture(stream)
    for t in range(max(lens)):
        plan.step_tokens([p[min(t, len(p) - 1)] for p in prompts], [min(t, len(p) - 1) for p in prompts], stream)
    theirs = plan.buffers.x.float().cpu().numpy()
    bridge.reset_graph()
    for i in range(3):
        norm_close(ours[i], theirs[i], 2e-2)
    for s in seqs:
        gen.cache.free(s)


def test_generate_mixes_prompts_and_forks(setup):
    from kudacuda_b200.paged_serving import Sampling

    _, _, gen = setup
    prompts = [prompt(n, 30 + n) for n in (100, 3, 20, 64)]
    greedy = gen.generate(prompts, 6)
    assert [len(a) for a in greedy] == [1] * 4 and all(len(a[0]) == 6 for a in greedy)
    assert gen.cache.free_pages == 64
    # the same first tokens whatever shares the steps (a near tie may fall either way)
    alone = [gen.generate([p], 1)[0][0][0] for p in prompts]
    assert sum(a[0][0] == b for a, b in zip(greedy, alone)) >= 3
    forked = gen.generate(prompts[2:3], 5, answers=3)[0]
    assert forked[1] == forked[2] and forked[0][0] == forked[1][0]
    drawn = gen.generate(prompts[:2], 8, Sampling(temperature=1.5, top_k=200, top_p=0.95, min_p=1e-4), answers=4, seed=3)
    again = gen.generate(prompts[:2], 8, Sampling(temperature=1.5, top_k=200, top_p=0.95, min_p=1e-4), answers=4, seed=3)
    assert drawn == again and len({tuple(a) for a in drawn[0]}) == 4
    assert gen.cache.free_pages == 64


def test_step_refuses(setup):
    from kudacuda_b200.paged_serving import PagedCacheFull, PagedSequence, Sampling

    _, _, gen = setup
    s = PagedSequence()
    with pytest.raises(ValueError):
        gen.step([], [], [])
    with pytest.raises(ValueError):
        gen.step([(s, [])], [Sampling()], [0.0])
    with pytest.raises(ValueError):
        gen.step([(s, [1] * 65)], [Sampling()], [0.0])
    with pytest.raises(ValueError):
        gen.step([(s, [1])], [], [0.0])
    with pytest.raises(PagedCacheFull):
        gen.cache.reserve([(s, 64 * 16 + 1)], 0)
    assert s.length == 0 and gen.cache.free_pages == 64


def test_cache_copies_on_another_stream(setup):
    """reserve and compact on a stream that is held up, while the current stream goes on taking memory."""

    from kudacuda_b200.paged_serving import PagedKVCache, PagedSequence

    bridge, _, _ = setup
    cache = PagedKVCache(bridge, layers=3, num_pages=24, kv_heads=2, head_dim=64, page_size=16, device=DEV)
    seqs = [PagedSequence() for _ in range(4)]
    cache.reserve([(s, 40) for s in seqs], 0)
    g = torch.Generator(device=DEV).manual_seed(3)
    cache.k.copy_(torch.randn(cache.k.shape, generator=g, device=DEV))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g, device=DEV))

    def contents(sequences):
        rows = []
        for s in sequences:
            pages = torch.tensor(s.pages, device=DEV)
            for x in (cache.k, cache.v):
                rows.append(x[:, pages].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :40].clone())
        return rows

    forks = [cache.fork(seqs[i]) for i in (1, 3)]
    alive = [seqs[1], seqs[3], *forks]
    want = contents(alive)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for what in ("reserve", "compact"):
        if what == "compact":
            cache.free(seqs[0])
            cache.free(seqs[2])
        table = torch.tensor(cache.table(alive), dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        if what == "reserve":
            cache.reserve([(f, 1) for f in forks], side.cuda_stream)
        else:
            assert cache.compact(alive, side.cuda_stream, block_table=table) > 0
        keep = [torch.full((n,), 5, dtype=torch.int32, device=DEV) for n in (1, 2, 4, 16, 24, 48) for _ in range(20)]
        torch.cuda.synchronize()
        assert bridge.error_word(clear=True) == 0 and keep
        assert all(torch.equal(x, y) for x, y in zip(contents(alive), want))
        if what == "compact":
            assert table.tolist() == cache.table(alive)


def test_step_refuses_a_sequence_named_twice(setup):
    from kudacuda_b200.paged_serving import PagedSequence, Sampling

    _, _, gen = setup
    s = PagedSequence()
    gen.step([(s, [3, 4])], [Sampling()], [0.0])
    with pytest.raises(ValueError, match="once"):
        gen.step([(s, [5]), (s, [6])], [Sampling()] * 2, [0.0] * 2)
    assert s.length == 2
    gen.cache.free(s)


def test_step_that_raises_can_be_taken_again(setup):
    """The settings of the last part of a step do not fit their type: the sequence is as it was before."""

    from kudacuda_b200.paged_serving import PagedSequence, Sampling

    _, _, gen = setup
    free = gen.cache.free_pages
    seq, other = PagedSequence(), PagedSequence()
    ids = prompt(33, 77)
    gen.step([(seq, ids[:20])], [Sampling()], [0.0])
    gen.step([(other, ids[:20])], [Sampling()], [0.0])
    with pytest.raises((RuntimeError, OverflowError, TypeError)):
        gen.step([(seq, ids[20:])], [Sampling(temperature=1.0, top_k=1 << 40)], [0.0])
    assert seq.length == 20 and gen.cache.free_pages == free - 4
    again, _ = gen.step([(seq, ids[20:])], [Sampling()], [0.0])
    x = gen.x[12].clone()
    first, _ = gen.step([(other, ids[20:])], [Sampling()], [0.0])
    assert again == first and torch.equal(gen.x[12], x)
    gen.cache.free(seq)
    gen.cache.free(other)


def test_generate_waits_for_pages(setup):
    """Prompts that do not fit together are served one after the other, as if each were alone."""

    from kudacuda_b200.paged_serving import PagedSequence

    _, _, gen = setup
    prompts = [prompt(n, 50 + n) for n in (33, 40, 16, 1)]
    held = PagedSequence()
    gen.cache.reserve([(held, 16 * 60)], torch.cuda.current_stream().cuda_stream)
    tight = gen.generate(prompts, 5)
    gen.cache.free(held)
    assert gen.cache.free_pages == 64 and [len(a[0]) for a in tight] == [5] * 4
    # (the first prompt is alone in its steps; a near tie may fall either way for the others)
    assert tight[0] == gen.generate(prompts[:1], 5)[0]
