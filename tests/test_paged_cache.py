"""CPU tests of the paged cache's host side: pages taken, shared, copied on write,
freed and compacted (the copies done by a stand-in for the bridge), rotary
tables, and the refusals of the bridge's paged methods before any native call."""

import math
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from kudacuda_b200.kudacuda_sidecar import KudaCudaBridge  # noqa: E402
from kudacuda_b200.paged_serving import (  # noqa: E402
    PagedCacheFull, PagedGenerator, PagedKVCache, PagedSequence, Sampling, paged_rope_tables)


class Copier:
    """What dispatch_kv_pages_copy does, on the CPU, with its condition checked."""

    def __init__(self):
        self.calls = []

    def dispatch_kv_pages_copy(self, k, v, pairs, *, stream_ptr, block_table=None, page_map=None):
        pairs = pairs.tolist()
        self.calls.append(pairs)
        assert not {a for a, _ in pairs} & {b for _, b in pairs}
        assert len({b for _, b in pairs}) == len(pairs)
        for a, b in pairs:
            k[:, b], v[:, b] = k[:, a], v[:, a]
        if block_table is not None:
            valid = block_table >= 0
            block_table[valid] = page_map[block_table[valid].long()]


def make(num_pages=10, page=16):
    copier = Copier()
    cache = PagedKVCache(copier, layers=2, num_pages=num_pages, kv_heads=1, head_dim=4, page_size=page,
                         dtype=torch.float32, device="cpu")
    return cache, copier


def write(cache, seq, start, marks):
    """Token ``start + i`` of a sequence is marks[i], in every layer."""

    for i, m in enumerate(marks):
        page, slot = seq.pages[(start + i) // cache.page_size], (start + i) % cache.page_size
        cache.k[:, page, :, slot] = m
        cache.v[:, page, :, slot] = -m


def read(cache, seq):
    out = []
    for i in range(seq.length):
        page, slot = seq.pages[i // cache.page_size], i % cache.page_size
        got = {float(x) for x in cache.k[:, page, :, slot].flatten()} | {-float(x) for x in cache.v[:, page, :, slot].flatten()}
        assert len(got) == 1
        out.append(got.pop())
    return out


def grow(cache, seq, marks):
    start = seq.length
    cache.reserve([(seq, len(marks))], 0)
    write(cache, seq, start, marks)


def test_pages_are_taken_as_a_sequence_grows_and_come_back():
    cache, copier = make()
    a = PagedSequence()
    grow(cache, a, range(1, 17))
    assert a.pages == [0] and cache.free_pages == 9
    grow(cache, a, [17])
    assert a.pages == [0, 1] and read(cache, a) == list(range(1, 18))
    cache.reserve([(a, 0)], 0)
    assert cache.table([a, PagedSequence()]) == [[0, 1], [-1, -1]]
    cache.truncate(a, 16)
    assert a.pages == [0] and cache.free_pages == 9
    cache.free(a)
    assert cache.free_pages == 10 and a.length == 0 and not copier.calls


def test_forks_share_pages_until_one_grows():
    cache, copier = make()
    a = PagedSequence()
    grow(cache, a, range(1, 22))  # one full page, one of five
    b, c = cache.fork(a), cache.fork(a)
    assert b.pages == a.pages and cache.free_pages == 8
    cache.reserve([(b, 1), (c, 1)], 0)  # both grow at once: two copies, a keeps the original
    assert len(copier.calls) == 1 and len(copier.calls[0]) == 2
    write(cache, b, 21, [100])
    write(cache, c, 21, [200])
    grow(cache, a, [300])
    assert len(copier.calls) == 1
    base = list(range(1, 22))
    assert read(cache, a) == base + [300] and read(cache, b) == base + [100] and read(cache, c) == base + [200]
    assert a.pages[0] == b.pages[0] == c.pages[0] and len({a.pages[1], b.pages[1], c.pages[1]}) == 3
    cache.free(a)
    assert read(cache, b) == base + [100]
    cache.free(b)
    cache.free(c)
    assert cache.free_pages == 10


def test_all_owners_of_a_shared_page_growing_leave_one_with_the_original():
    cache, copier = make()
    a = PagedSequence()
    grow(cache, a, range(5))
    b = cache.fork(a)
    cache.reserve([(a, 1), (b, 1)], 0)
    assert len(copier.calls[0]) == 1 and a.pages != b.pages and cache.free_pages == 8


@pytest.mark.parametrize("owners,tokens", [(2, 1), (3, 1), (4, 12)])
def test_all_owners_grow_into_exactly_the_free_pages(owners, tokens):
    # each but one copies the page of five tokens; 12 more also start a page each
    need = owners - 1 + (owners if tokens > 11 else 0)
    cache, copier = make(num_pages=1 + need)
    a = PagedSequence()
    grow(cache, a, range(5))
    seqs = [a] + [cache.fork(a) for _ in range(owners - 1)]
    cache.reserve([(s, tokens) for s in seqs], 0)
    assert cache.free_pages == 0 and len(copier.calls[0]) == owners - 1
    assert len({p for s in seqs for p in s.pages}) == 1 + need
    assert all(read(cache, s)[:5] == list(range(5)) for s in seqs)
    for s in seqs:
        cache.free(s)
    assert cache.free_pages == 1 + need


def test_one_page_too_few_for_all_owners_changes_nothing():
    cache, copier = make(num_pages=2)
    a = PagedSequence()
    grow(cache, a, range(5))
    seqs = [a, cache.fork(a), cache.fork(a)]
    with pytest.raises(PagedCacheFull, match="2 pages are needed, 1 are free"):
        cache.reserve([(s, 1) for s in seqs], 0)
    assert all(s.pages == [0] and s.length == 5 for s in seqs) and cache.free_pages == 1 and not copier.calls
    with pytest.raises(PagedCacheFull):
        cache.reserve([(s, 1) for s in seqs[:2]], 0)  # the third keeps the original, so both copy
    cache.reserve([(seqs[0], 1)], 0)
    assert cache.free_pages == 0


def test_a_fork_of_whole_pages_copies_nothing():
    cache, copier = make()
    a = PagedSequence()
    grow(cache, a, range(32))
    b = cache.fork(a)
    grow(cache, b, [7])
    assert not copier.calls and b.pages[:2] == a.pages and read(cache, b) == [*map(float, range(32)), 7.0]


def test_a_full_cache_refuses_and_changes_nothing():
    cache, _ = make(num_pages=3)
    a, b = PagedSequence(), PagedSequence()
    grow(cache, a, range(20))
    with pytest.raises(PagedCacheFull):
        cache.reserve([(a, 1), (b, 17)], 0)
    assert a.length == 20 and b.length == 0 and not b.pages and cache.free_pages == 1
    f = cache.fork(a)
    with pytest.raises(PagedCacheFull):
        cache.reserve([(f, 13)], 0)  # its copy of the shared page and one more
    assert f.pages == a.pages and f.length == 20
    with pytest.raises(ValueError):
        cache.reserve([(a, -1)], 0)
    with pytest.raises(ValueError):
        cache.truncate(a, 21)


def test_a_copy_that_fails_changes_nothing():
    cache, copier = make()
    a = PagedSequence()
    grow(cache, a, range(5))
    b = cache.fork(a)

    def fail(*args, **kw):
        raise RuntimeError("no copy")

    copier.dispatch_kv_pages_copy = fail
    with pytest.raises(RuntimeError, match="no copy"):
        cache.reserve([(a, 30), (b, 1)], 0)
    assert a.pages == b.pages == [0] and a.length == b.length == 5 and cache.free_pages == 9
    cache.free(a)
    cache.free(b)
    assert cache.free_pages == 10


def test_a_step_that_raises_leaves_its_sequences_as_they_were():
    cache, copier = make()
    gen = PagedGenerator.__new__(PagedGenerator)
    gen.torch = StreamedTorch()
    gen.cache, gen.device, gen.cos = cache, "cpu", torch.zeros((100, 2))
    gen.config = SimpleNamespace(layers=0, hidden=4, vocab=9, eps=1e-6)
    gen.weights = SimpleNamespace(layers=[], embedding=None)
    gen.q = gen.attn = gen.qkv_out = gen.x = torch.zeros((64, 4))
    done = []

    def fail(*args, **kw):
        raise RuntimeError("no embedding")

    gen.bridge = SimpleNamespace(dispatch_batch_embedding=fail)
    a = PagedSequence()
    grow(cache, a, range(20))
    b = cache.fork(a)
    stream = SimpleNamespace(cuda_stream=0, synchronize=lambda: done.append(1))
    with pytest.raises(RuntimeError, match="no embedding"):
        gen.step([(a, [1] * 30), (b, [2]), (PagedSequence(), [3])], [Sampling()] * 3, [0.5] * 3, stream)
    # (one of the two owners may keep its copy of the page they shared)
    assert a.length == b.length == 20 and len(a.pages) == len(b.pages) == 2 and cache.free_pages >= 7 and done
    assert read(cache, a) == read(cache, b) == list(range(20))
    cache.free(a)
    cache.free(b)
    assert cache.free_pages == 10


class Counting(PagedGenerator):
    """A generator whose steps only take pages; the token drawn is the sequence's length."""

    def __init__(self, num_pages, page=16):
        self.cache, self.copier = make(num_pages, page)
        self.steps, self.least = 0, num_pages

    def step(self, entries, sampling, uniform, stream=None):
        self.cache.reserve([(s, len(t)) for s, t in entries], 0)
        self.steps += 1
        self.least = min(self.least, self.cache.free_pages)
        return [s.length for s, _ in entries], [0.0] * len(entries)


@pytest.mark.parametrize("pages,lengths,new,answers", [
    (4, [16] * 5, 5, 1), (3, [1, 33, 2, 40], 8, 1), (10, [16, 17, 15, 1, 31], 20, 3), (40, [100, 200, 7], 50, 4),
    (5, [64, 64, 10], 17, 1), (7, [33, 16], 1, 5),
])
def test_prompts_wait_until_their_pages_are_free(pages, lengths, new, answers):
    gen = Counting(pages)
    out = gen.generate([[1] * n for n in lengths], new, answers=answers)
    assert out == [[[n + t for t in range(new)]] * answers for n in lengths]
    assert gen.cache.free_pages == pages


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 50])
@pytest.mark.parametrize("new", [1, 2, 15, 16, 17, 40])
@pytest.mark.parametrize("answers", [1, 2, 5])
def test_pages_of_a_prompt_and_its_answers(length, new, answers):
    gen = Counting(100)
    gen.generate([[1] * length], new, answers=answers)
    most = gen._most_pages(length, new, answers)
    assert 100 - gen.least == most
    Counting(most).generate([[1] * length], new, answers=answers)
    with pytest.raises(PagedCacheFull):  # one alone that does not fit is refused, and leaves nothing behind
        gen = Counting(most)
        held = PagedSequence()
        gen.cache.reserve([(held, 1)], 0)
        gen.generate([[1] * length], new, answers=answers)
    assert gen.cache.free_pages == most - 1


def test_prompts_that_fit_together_share_steps():
    gen = Counting(100)
    gen.generate([[1] * 10] * 5, 6)
    assert gen.steps == 6


def test_a_sequence_named_twice_is_refused():
    """Both entries would get the length with all tokens, and write the same place."""

    cache, copier = make()
    a, b = PagedSequence(), PagedSequence()
    grow(cache, a, range(3))
    with pytest.raises(ValueError, match="once"):
        cache.reserve([(a, 1), (b, 2), (a, 1)], 0)
    assert a.length == 3 and b.length == 0 and a.pages == [0] and cache.free_pages == 9 and not copier.calls
    cache.reserve([(a, 1), (cache.fork(a), 1), (b, 2)], 0)  # equal, but another sequence


def test_compaction_keeps_every_sequence_and_rewrites_tables():
    cache, copier = make(num_pages=12)
    seqs = [PagedSequence() for _ in range(4)]
    for i, s in enumerate(seqs):
        grow(cache, s, [100 * i + j for j in range(40)])
    fork = cache.fork(seqs[3])
    cache.free(seqs[0])
    cache.free(seqs[2])
    alive = [seqs[1], seqs[3], fork]
    want = [read(cache, s) for s in alive]
    table = torch.tensor(cache.table(alive), dtype=torch.int32)
    moved = cache.compact(alive, 0, block_table=table)
    assert moved == 3 and [read(cache, s) for s in alive] == want
    assert sorted({p for s in alive for p in s.pages}) == list(range(6))
    assert table.tolist() == cache.table(alive)
    assert cache.free_pages == 6 and cache.compact(alive, 0) == 0
    with pytest.raises(ValueError):
        cache.compact(alive[:1], 0)
    grow(cache, fork, [9])
    assert read(cache, seqs[3]) == want[1] and read(cache, fork) == want[2] + [9]
    for s in alive:
        cache.free(s)
    assert cache.free_pages == 12


class StreamedTorch:
    """torch whose tensors stay on the host; notes which stream is current as each one is made."""

    def __init__(self):
        self.current, self.made = 7, []
        self.cuda = SimpleNamespace(ExternalStream=lambda ptr, device=None: ptr, stream=self._use)

    def _use(self, stream):
        import contextlib

        @contextlib.contextmanager
        def use():
            self.current, before = stream, self.current
            try:
                yield
            finally:
                self.current = before

        return use()

    def _maker(self, make):
        def made(*args, device=None, **kw):
            out = make(*args, **kw)
            self.made.append((self.current, out.data_ptr()))
            return out
        return made

    def __getattr__(self, name):
        value = getattr(torch, name)
        return self._maker(value) if name in ("tensor", "arange", "zeros") else value


def test_compaction_needs_the_forks_too():
    cache, copier = make()
    a, b = PagedSequence(), PagedSequence()
    grow(cache, a, range(20))
    grow(cache, b, range(100, 120))
    fork = cache.fork(b)
    cache.free(a)
    with pytest.raises(ValueError, match="all of the cache's sequences"):
        cache.compact([b], 0)  # its pages are all that are in use, but the fork would be left behind
    assert b.pages == fork.pages == [2, 3] and not copier.calls
    assert cache.compact([b, fork, b], 0) == 2 and b.pages == fork.pages == [0, 1]
    assert read(cache, b) == read(cache, fork) == list(range(100, 120))


def test_copies_use_memory_of_the_stream_they_run_on():
    """The lists of a copy go back to the allocator as soon as it is launched, so they must come from the
    stream that it runs on: another one could take their memory while the copy still reads them."""

    class Streamed(Copier):
        def dispatch_kv_pages_copy(self, k, v, pairs, *, stream_ptr, block_table=None, page_map=None):
            lists = [t.data_ptr() for t in (pairs, page_map) if t is not None]
            streams.append([{p: s for s, p in fake.made}[p] for p in lists])
            assert stream_ptr == 99
            super().dispatch_kv_pages_copy(k, v, pairs, stream_ptr=stream_ptr, block_table=block_table, page_map=page_map)

    fake, streams = StreamedTorch(), []
    cache = PagedKVCache(Streamed(), layers=1, num_pages=8, kv_heads=1, head_dim=4, page_size=16, dtype=torch.float32,
                         device="cuda:0", torch_module=fake)
    a, b = PagedSequence(), PagedSequence()
    cache.reserve([(a, 5), (b, 40)], 99)
    f = cache.fork(b)
    cache.reserve([(f, 1)], 99)
    assert streams == [[99]]
    cache.free(a)
    table = torch.tensor(cache.table([b, f]), dtype=torch.int32)
    assert cache.compact([b, f], 99, block_table=table) == 1
    assert streams == [[99], [99, 99]] and table.tolist() == cache.table([b, f])


def test_rope_tables():
    cos, sin = paged_rope_tables(40, 64, 1e4)
    i, pos = 7, 33
    angle = pos * 1e4 ** (-2 * i / 64)
    assert abs(float(cos[pos, i]) - math.cos(angle)) < 1e-7 and abs(float(sin[pos, i]) - math.sin(angle)) < 1e-7
    lin, _ = paged_rope_tables(40, 64, 1e4, {"type": "linear", "factor": 4.0})
    assert torch.equal(lin[32], cos[8])  # positions counted in quarters
    ntk, _ = paged_rope_tables(40, 64, 1e4, {"type": "ntk", "factor": 4.0})
    assert torch.equal(ntk[:, 0], cos[:, 0])  # the fastest pair as it was, the slowest as with linear
    assert abs(math.acos(float(ntk[39, 31])) * 4 - math.acos(float(cos[39, 31]))) < 1e-3
    setting = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original": 8192}
    l3, _ = paged_rope_tables(5000, 128, 5e5, setting)
    plain, _ = paged_rope_tables(5000, 128, 5e5)
    assert torch.equal(l3[:, 0], plain[:, 0])
    slow = 4999 * 5e5 ** (-126 / 128)
    assert abs(float(l3[4999, 63]) - math.cos(slow / 8)) < 1e-6
    yarn, _ = paged_rope_tables(64, 128, 1e4, {"type": "yarn", "factor": 4.0, "original": 4096})
    gain = 0.1 * math.log(4.0) + 1
    assert abs(float(yarn[0, 5]) - gain) < 1e-6 and abs(float(yarn[5, 0]) - gain * math.cos(5)) < 1e-6
    assert abs(float(yarn[63, 63]) - gain * math.cos(63 * 1e4 ** (-126 / 128) / 4)) < 1e-6
    with pytest.raises(ValueError):
        paged_rope_tables(4, 3, 1e4)
    with pytest.raises(ValueError):
        paged_rope_tables(4, 4, 1e4, {"type": "other"})


# ------------------------------------------------------------------ the bridge's checks
class Recorder:
    """Stands for the library: every entry succeeds and is noted."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if not name.startswith("kudacuda_"):
            raise AttributeError(name)

        def entry(*args):
            self.calls.append((name, args))
            return 1 if name == "kudacuda_create" else 4096 if name.endswith("_bytes") else 0

        return entry


@pytest.fixture()
def bridge():
    lib = Recorder()
    br = KudaCudaBridge(device_id=0, native_lib=lib)
    br.device_id = -1  # the index that torch gives host memory
    lib.calls.clear()
    yield SimpleNamespace(br=br, lib=lib)


BF16 = torch.bfloat16


def attention_args(**kw):
    a = dict(query=torch.zeros((3, 4, 64), dtype=BF16), k=torch.zeros((6, 2, 16, 64), dtype=BF16),
             v=torch.zeros((6, 2, 16, 64), dtype=BF16), out=torch.zeros((3, 4, 64), dtype=BF16),
             start=torch.zeros(3, dtype=torch.int32), kv=torch.zeros(2, dtype=torch.int32),
             table=torch.zeros((2, 5), dtype=torch.int32), ws=torch.zeros(4096, dtype=torch.uint8), lse=None)
    return a | kw


def attend(br, a):
    br.dispatch_paged_attention(a["query"], a["k"], a["v"], a["out"], a["start"], a["kv"], a["table"], a["ws"],
                                max_query=2, lse=a["lse"], stream_ptr=-1)


def test_paged_attention_passes_shapes_strides_and_types(bridge):
    wide = torch.zeros((3, 600), dtype=torch.float16)
    f16 = dict(query=wide[:, 40:296].view(3, 4, 64), out=torch.zeros((3, 256), dtype=torch.float16),
               k=torch.zeros((6, 2, 16, 64), dtype=torch.float16), v=torch.zeros((6, 2, 16, 64), dtype=torch.float16),
               table=torch.zeros((2, 9), dtype=torch.int32)[:, 2:7])
    a = attention_args(**f16)
    attend(bridge.br, a)
    name, args = bridge.lib.calls[-1]
    assert name == "kudacuda_sm100_paged_attention"
    assert args[1] == 1 and args[3] == 600 and args[7] == 256 and args[10] == 4096
    assert args[14:24] == (9, 5, 2, 3, 2, 4, 2, 64, 6, 16) and args[24] == 0.125
    assert args[25] == 0xFFFFFFFFFFFFFFFF
    attend(bridge.br, attention_args())
    assert bridge.lib.calls[-1][1][1] == 2


@pytest.mark.parametrize("kw", [
    dict(query=torch.zeros((3, 4, 64))), dict(query=torch.zeros((3, 4, 64), dtype=torch.float16)),
    dict(query=torch.zeros((3, 64, 4), dtype=BF16).transpose(1, 2)), dict(query=torch.zeros((12, 64), dtype=BF16)[:, ::2]),
    dict(out=torch.zeros((2, 4, 64), dtype=BF16)), dict(out=torch.zeros((3, 4, 64), dtype=torch.float16)),
    dict(k=torch.zeros((6, 2, 16, 128), dtype=BF16)), dict(k=torch.zeros((2, 16, 64), dtype=BF16)),
    dict(k=torch.zeros((6, 16, 2, 64), dtype=BF16).transpose(1, 2)), dict(table=torch.zeros((2, 5))),
    dict(table=torch.zeros((5, 2), dtype=torch.int32).t()), dict(start=torch.zeros(2, dtype=torch.int32)),
    dict(start=torch.zeros(3)), dict(kv=torch.zeros(1, dtype=torch.int32)), dict(kv=torch.zeros(4, dtype=torch.int32)[::2]),
    dict(lse=torch.zeros((3, 2))), dict(lse=torch.zeros((3, 4), dtype=BF16)),
])
def test_paged_attention_refuses(bridge, kw):
    with pytest.raises(ValueError):
        attend(bridge.br, attention_args(**kw))
    assert not bridge.lib.calls


def test_paged_attention_refuses_a_workspace_smaller_than_it_says(bridge):
    with pytest.raises(ValueError, match="workspace"):
        attend(bridge.br, attention_args(ws=torch.zeros(1, dtype=torch.uint8).expand(4096)))
    assert not bridge.lib.calls


def append_args(**kw):
    a = dict(qkv=torch.zeros((3, 8 * 64), dtype=BF16), q=torch.zeros((3, 4, 64), dtype=BF16),
             cos=torch.zeros((9, 16)), sin=torch.zeros((9, 16)), bias=None)
    return attention_args() | a | kw


def append(br, a):
    br.dispatch_rope_append_paged(a["qkv"], a["q"], a["k"], a["v"], a["cos"], a["sin"], a["start"], a["kv"], a["table"],
                                  interleaved=True, bias=a["bias"], stream_ptr=3)


def test_rope_append_passes_shapes_and_takes_no_tables(bridge):
    append(bridge.br, append_args(bias=torch.zeros(512, dtype=BF16)))
    name, args = bridge.lib.calls[-1]
    assert name == "kudacuda_sm100_rope_append_paged" and args[1] == 2 and args[3] == 512 and args[6] == 256
    assert args[11:14] == (9, 32, 1) and args[17:26] == (5, 5, 2, 3, 4, 2, 64, 6, 16) and args[26] == 3
    append(bridge.br, append_args(cos=None, sin=None))
    assert bridge.lib.calls[-1][1][9:14] == (0, 0, 0, 0, 1)


@pytest.mark.parametrize("kw", [
    dict(qkv=torch.zeros((3, 7 * 64), dtype=BF16)), dict(qkv=torch.zeros((3, 8 * 64))),
    dict(q=torch.zeros((4, 4, 64), dtype=BF16)), dict(cos=torch.zeros((9, 16), dtype=BF16)),
    dict(sin=torch.zeros((8, 16))), dict(cos=torch.zeros((16, 9)).t(), sin=torch.zeros((16, 9)).t()),
    dict(bias=torch.zeros(511, dtype=BF16)), dict(bias=torch.zeros(512)),
])
def test_rope_append_refuses(bridge, kw):
    with pytest.raises(ValueError):
        append(bridge.br, append_args(**kw))
    assert not bridge.lib.calls


@pytest.mark.parametrize("kw", [dict(cos=None), dict(sin=None)])
def test_rope_append_refuses_one_table_without_the_other(bridge, kw):
    with pytest.raises(ValueError, match="together"):
        append(bridge.br, append_args(**kw))
    assert not bridge.lib.calls


def test_pages_copy_passes_and_refuses(bridge):
    k, v = torch.zeros((3, 7, 2, 16, 8), dtype=BF16), torch.zeros((3, 7, 2, 16, 8), dtype=BF16)
    pairs = torch.zeros((2, 2), dtype=torch.int32)
    table, page_map = torch.zeros((4, 9), dtype=torch.int32)[:, 1:6], torch.zeros(7, dtype=torch.int32)
    bridge.br.dispatch_kv_pages_copy(k, v, pairs, block_table=table, page_map=page_map, stream_ptr=0)
    args = bridge.lib.calls[-1][1]
    assert args[3:7] == (3, 7 * 512, 7, 512) and args[8] == 2 and args[10:13] == (9, 4, 5)
    bridge.lib.calls.clear()
    for kw in (dict(block_table=table), dict(page_map=page_map), dict(block_table=table, page_map=page_map[:6]),
               dict(block_table=table.long(), page_map=page_map)):
        with pytest.raises(ValueError):
            bridge.br.dispatch_kv_pages_copy(k, v, pairs, stream_ptr=0, **kw)
    for bad in ((k, v[:2], pairs), (k, v.float(), pairs), (k, v, pairs.long()), (k, v, pairs[:, :1]),
                (k[:, ::2], v[:, ::2], pairs), (k[0, 0, 0], v[0, 0, 0], pairs)):
        with pytest.raises(ValueError):
            bridge.br.dispatch_kv_pages_copy(*bad, stream_ptr=0)
    assert not bridge.lib.calls


def test_pages_copy_of_one_layer_goes_by_its_shape(bridge):
    """The stride of the single layer is a page's; the tensor is contiguous all the same."""

    k, v = (torch.zeros((4, 1, 2, 16, 64), dtype=BF16).transpose(0, 1) for _ in range(2))
    assert k.is_contiguous() and k.stride(0) == 2048
    bridge.br.dispatch_kv_pages_copy(k, v, torch.zeros((1, 2), dtype=torch.int32), stream_ptr=0)
    assert bridge.lib.calls[-1][1][3:7] == (1, 4 * 4096, 4, 4096)


def test_sample_passes_and_refuses(bridge):
    x, u, tok = torch.zeros((3, 20), dtype=BF16)[:, 4:14], torch.zeros(3), torch.zeros(3, dtype=torch.int32)
    bridge.br.dispatch_sample(x, tok, u, top_k=tok, stream_ptr=0)
    args = bridge.lib.calls[-1][1]
    assert args[1] == 2 and args[3:6] == (20, 3, 10) and args[6] == 0 and args[7] != 0 and args[8] == args[9] == 0
    bridge.lib.calls.clear()
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=torch.zeros((10, 3)).t()), dict(tokens=tok.long()),
                dict(tokens=tok[:2]), dict(uniform=u.double()), dict(temperature=tok), dict(top_k=u), dict(top_p=u[:1]),
                dict(min_p=torch.zeros(6)[::2]), dict(logprobs=u.half())):
        a = dict(logits=x, tokens=tok, uniform=u) | bad
        with pytest.raises(ValueError):
            bridge.br.dispatch_sample(a.pop("logits"), a.pop("tokens"), a.pop("uniform"), stream_ptr=0, **a)
    assert not bridge.lib.calls
