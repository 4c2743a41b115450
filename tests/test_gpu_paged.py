"""GPU parity of the paged-cache operators and of sampling against plain
64-bit statements (tests/paged_reference.py).

Tolerances, with u half of the type's spacing at 1 (2^-8 bf16, 2^-11 f16):
* attention: the output is rounded once (u |o|) and the probabilities that
  multiply V may be rounded once each (u sum p |v|); 32-bit scores, sums and
  exponentials add at most 2^-14 sum p |v|.  lse: the scores are 32-bit sums of
  head_dim products (head_dim 2^-24 sum |q k| scale) plus 2^-18.
* rotary: one rounding (u |y|) and three 32-bit operations (2^-22 (|x0| + |x1|)).
* copies and appended values are exact; sampled tokens are equal (the 32-bit
  exponentials move a boundary by about 1e-6 of the mass, so one of the few
  hundred fixed draws meets one with probability about 1e-3), log-probabilities
  within 2^-16 (argument rounding |z| 2^-23, z below 40, and its sum).
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from tests import paged_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def bridge():
    from kudacuda_b200.kudacuda_sidecar import KudaCudaBridge

    torch.cuda.set_device(0)
    br = KudaCudaBridge(device_id=0)
    yield br
    br.shutdown()


def attend(bridge, q, k, v, table, new, lens, *, scale=None, max_query=None, out=None, stream=None):
    rows, heads, d = q.shape
    start = R.starts(new, DEV)
    kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if out is None:
        out = torch.full((rows, heads, d), 7.0, dtype=q.dtype, device=DEV)
    lse = torch.full((rows, heads), 7.0, dtype=torch.float32, device=DEV)
    most = max(new) if max_query is None else max_query
    ws = bridge.paged_attention_workspace(q, k, table, max_query=most)
    ws.fill_(0xA5)  # its contents need no initialisation
    torch.cuda.synchronize()
    bridge.dispatch_paged_attention(q, k, v, out, start, kv, table, ws, max_query=most, lse=lse, scale=scale,
                                    stream_ptr=int((stream or torch.cuda.current_stream()).cuda_stream))
    torch.cuda.synchronize()
    return out, lse


def check_attention(q, new, lens, keys, vals, out, lse, scale):
    d = q.shape[-1]
    ref, ref_lse, mag, reach = R.attention(q.cpu(), new, lens, keys, vals, scale)
    u = R.UNIT[q.dtype]
    got, got_lse = out.double().cpu(), lse.double().cpu()
    bound = u * ref.abs() + (u + 2.0**-14) * mag
    assert torch.isfinite(got).all()
    bad = (got - ref).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} outputs off, first at {bad.nonzero()[0].tolist()}"
    empty = ref_lse == -math.inf
    assert torch.equal(got_lse == -math.inf, empty)
    assert (got[empty] == 0).all()
    lse_bound = d * 2.0**-24 * reach + 2.0**-18
    diff = torch.where(empty, torch.zeros_like(ref_lse), got_lse - ref_lse).abs()
    assert (diff <= lse_bound).all(), f"lse off by {float((diff - lse_bound).max())} over its bound"


ATTENTION = [
    # dtype, q_heads, kv_heads, d, page, new tokens, lengths with them
    (BF16, 16, 2, 128, 16, [1], [1]),
    (BF16, 16, 2, 128, 16, [1], [509]),
    (F16, 32, 8, 128, 64, [1, 1, 1], [17, 128, 1000]),
    (BF16, 16, 2, 128, 32, [1, 1, 0, 1, 1], [0, 5, 33, 2048, 64]),   # an empty sequence, one without new tokens
    (BF16, 5, 5, 64, 16, [1, 2, 3], [100, 2, 3]),
    (F16, 7, 1, 64, 128, [1, 1], [300, 129]),
    (BF16, 28, 4, 128, 16, [3, 1, 5], [257, 600, 5]),
    (BF16, 16, 2, 128, 64, [4, 2, 9], [1, 2, 400]),                  # more new tokens than the length: empty rows
    (BF16, 8, 1, 128, 128, [130], [130]),
    (F16, 32, 8, 128, 16, [77, 1, 31], [77, 333, 200]),
    (BF16, 2, 2, 64, 32, [65, 200], [129, 260]),
    (BF16, 15, 3, 128, 16, [40, 0, 27], [50, 10, 411]),              # five heads a group
    (F16, 24, 2, 64, 16, [19, 33], [97, 64]),                        # twelve heads a group
    (BF16, 40, 1, 128, 64, [7, 11], [70, 300]),                      # forty heads of one key head
    (BF16, 16, 16, 128, 64, [129], [515]),
    (BF16, 4, 1, 128, 64, [300, 1, 60], [1100, 900, 60]),
    (F16, 160, 1, 64, 16, [2, 1], [40, 19]),                         # more heads a group than a tile has rows
]


@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention_against_64_bits(bridge, case):
    dtype, qh, kh, d, page, new, lens = ATTENTION[case]
    k, v, table, keys, vals = R.make_cache(lens, kh, page, d, dtype, DEV, 100 + case)
    g = torch.Generator().manual_seed(200 + case)
    q = (1.5 * torch.randn((sum(new), qh, d), generator=g)).to(dtype).to(DEV)
    out, lse = attend(bridge, q, k, v, table, new, lens)
    assert bridge.error_word(clear=True) == 0
    check_attention(q, new, lens, keys, vals, out, lse, 1 / math.sqrt(d))


@pytest.mark.parametrize("new,lens", [([1, 1], [5000, 9001]), ([70], [3000])])
def test_attention_scores_far_apart(bridge, new, lens):
    """Scores to hundreds, the largest at the far end: the running maximum moves late."""

    dtype, qh, kh, d, page = BF16, 8, 2, 128, 64
    k, v, table, keys, vals = R.make_cache(lens, kh, page, d, dtype, DEV, 31)
    for b, n in enumerate(lens):  # keys that grow along the sequence
        gain = torch.linspace(0.1, 6.0, n, dtype=torch.float64)[None, :, None]
        keys[b] = (keys[b] * gain).to(dtype).double()
        for j in range((n + page - 1) // page):
            m = min(page, n - j * page)
            k[table[b, j], :, :m] = keys[b][:, j * page:j * page + m].to(dtype).to(DEV)
    g = torch.Generator().manual_seed(32)
    q = (3.0 * torch.randn((sum(new), qh, d), generator=g)).to(dtype).to(DEV)
    out, lse = attend(bridge, q, k, v, table, new, lens)
    assert bridge.error_word(clear=True) == 0
    check_attention(q, new, lens, keys, vals, out, lse, 1 / math.sqrt(d))


def small_weights(bridge, dtype, heads, below, step, n=20_032, d=64):
    """The first key takes almost all of the weight but its value is 0: the output is that of the others, each
    ``below`` nats less.  As many equal sequences as the device has SMs, so that one running maximum goes
    through a sequence's whole length.  ``step``: half of the spacing of the smallest f16 weights, as a part
    of the largest weight, by which each may be off beside its rounding (bf16 has no such end)."""

    g = torch.Generator().manual_seed(int(10 * below) + heads)
    kk = (0.01 * torch.randn((1, n, d), generator=g)).to(dtype)
    vv = (64 * (0.5 + torch.rand((1, n, d), generator=g))).to(dtype)
    kk[:, 0, :] = 0
    kk[:, :, 0] = 0
    kk[:, 0, 0] = 8.0
    vv[:, 0] = 0
    q = 0.3 * torch.randn((1, heads, d), generator=g)
    q[:, :, 0] = below * math.sqrt(d) / 8.0
    q = q.to(dtype)
    batch = torch.cuda.get_device_properties(0).multi_processor_count
    k, v = (x.view(n // 64, 1, 64, d).to(DEV) for x in (kk, vv))
    table = torch.arange(n // 64, dtype=torch.int32, device=DEV).repeat(batch, 1)
    out, _ = attend(bridge, q.to(DEV).repeat(batch, 1, 1), k, v, table, [1] * batch, [n] * batch)
    assert bridge.error_word(clear=True) == 0
    ref, _, mag, _ = R.attention(q, [1], [n], [kk.double()], [vv.double()], 1 / math.sqrt(d))
    u = R.UNIT[dtype]
    bound = u * ref.abs() + (u + 2.0**-14) * mag + (n * step * 96 + 2.0**-25 if dtype == F16 else 0)
    for r in (0, 1, batch // 2, batch - 1):
        worst = ((out[r:r + 1].double().cpu() - ref).abs() / bound).max()
        assert worst <= 1, f"{float(worst)} of the bound"


@pytest.mark.parametrize("dtype,heads", [(F16, 1), (BF16, 1), (F16, 12)])
@pytest.mark.parametrize("below", [12.0, 17.4, 19.0])
def test_attention_small_weights_beside_a_large_one(bridge, dtype, heads, below):
    small_weights(bridge, dtype, heads, below, 2.0**-40)


@pytest.mark.parametrize("dtype,heads", [(F16, 32), (BF16, 32), (F16, 17)])
@pytest.mark.parametrize("below", [12.0, 17.4, 19.0])
def test_attention_small_weights_with_many_rows(bridge, dtype, heads, below):
    small_weights(bridge, dtype, heads, below, 2.0**-36)


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [70, 300, 129]), ([90, 3], [200, 77])])
def test_attention_strided_rows_scale_stream_and_wide_table(bridge, new, lens):
    """Rows that are a slice of a wider buffer, a table that is a slice of a wider one, a scale of the
    caller's, a stream other than the current one, no lse."""

    dtype, qh, kh, d, page = BF16, 16, 2, 128, 16
    k, v, table, keys, vals = R.make_cache(lens, kh, page, d, dtype, DEV, 41, width=40)
    wide = torch.full((len(lens), 57), 999999, dtype=torch.int32, device=DEV)
    wide[:, 8:48] = table
    g = torch.Generator().manual_seed(42)
    rows = sum(new)
    full = torch.randn((rows, (qh + 2 * kh) * d), generator=g).to(dtype).to(DEV)
    q = full[:, :qh * d].view(rows, qh, d)
    canvas = torch.full((rows, 3 * qh * d), 5.0, dtype=dtype, device=DEV)
    out = canvas[:, qh * d:2 * qh * d].unflatten(1, (qh, d))
    stream = torch.cuda.Stream()
    got, lse = attend(bridge, q, k, v, wide[:, 8:48], new, lens, scale=0.2, out=out, stream=stream)
    assert bridge.error_word(clear=True) == 0
    check_attention(q, new, lens, keys, vals, got, lse, 0.2)
    assert (canvas[:, :qh * d] == 5.0).all() and (canvas[:, 2 * qh * d:] == 5.0).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [60, 1, 17]])
def test_attention_does_not_depend_on_the_batch_and_repeats(bridge, new):
    """A second run gives the same bits, and a graph replay too."""

    lens = [600, 77, 1500]
    k, v, table, keys, vals = R.make_cache(lens, 8, 32, 128, F16, DEV, 51)
    q = torch.randn((sum(new), 32, 128), generator=torch.Generator().manual_seed(52)).to(F16).to(DEV)
    first, lse1 = attend(bridge, q, k, v, table, new, lens)
    second, lse2 = attend(bridge, q, k, v, table, new, lens)
    assert torch.equal(first, second) and torch.equal(lse1, lse2)
    start, kv = R.starts(new, DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.zeros_like(first)
    ws = bridge.paged_attention_workspace(q, k, table, max_query=max(new))
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        bridge.dispatch_paged_attention(q, k, v, out, start, kv, table, ws, max_query=max(new),
                                        stream_ptr=int(torch.cuda.current_stream().cuda_stream))
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    # lengths are device data: the same graph serves shorter ones
    shorter = [300, 70, 1201]
    kv.copy_(torch.tensor(shorter, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want, _ = attend(bridge, q, k, v, table, new, shorter)
    assert torch.equal(out, want)
    assert bridge.error_word(clear=True) == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new,lens,heads,kv_heads", [([1, 70, 3], [900, 333, 40], 16, 2), ([300, 1], [300, 4000], 4, 1)])
def test_attention_with_a_smaller_max_query_keeps_the_probabilities(bridge, dtype, new, lens, heads, kv_heads):
    """The kernel that max_query = 1 chooses takes any number of rows, and rounds the output alone to the type."""

    k, v, table, keys, vals = R.make_cache(lens, kv_heads, 32, 128, dtype, DEV, 57)
    q = torch.randn((sum(new), heads, 128), generator=torch.Generator().manual_seed(58)).to(dtype)
    out, lse = attend(bridge, q.to(DEV), k, v, table, new, lens, max_query=1)
    assert bridge.error_word(clear=True) == 0
    check_attention(q, new, lens, keys, vals, out, lse, 128**-0.5)
    ref, _, mag, _ = R.attention(q, new, lens, keys, vals, 128**-0.5)
    assert ((out.double().cpu() - ref).abs() <= R.UNIT[dtype] * ref.abs() + 2.0**-14 * mag).all()


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [60, 1, 17, 1], [3, 1, 200, 2]])
def test_attention_of_a_part_of_the_batch(bridge, new):
    """Sequences alone, in twos and all together give the same rows, within the bound of either."""

    lens = [600, 77, 1500, 300]
    k, v, table, keys, vals = R.make_cache(lens, 2, 32, 128, BF16, DEV, 53)
    q = torch.randn((sum(new), 16, 128), generator=torch.Generator().manual_seed(54)).to(BF16).to(DEV)
    at = [sum(new[:i]) for i in range(5)]
    for part in ([0], [1], [2], [3], [0, 1], [1, 3], [2, 3], [0, 1, 2, 3]):
        rows = torch.cat([q[at[i]:at[i + 1]] for i in part])
        some = [[x[i] for i in part] for x in (new, lens, keys, vals)]
        out, lse = attend(bridge, rows, k, v, table[part], some[0], some[1])
        assert bridge.error_word(clear=True) == 0
        check_attention(rows, *some, out, lse, 128**-0.5)


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_attention_flags_a_missing_page_and_spares_the_others(bridge, new):
    lens = [200, 150]
    k, v, table, keys, vals = R.make_cache(lens, 2, 16, 128, BF16, DEV, 61, junk=0.0)
    q = torch.randn((sum(new), 16, 128), generator=torch.Generator().manual_seed(62)).to(BF16).to(DEV)
    good, _ = attend(bridge, q, k, v, table, new, lens)
    broken = table.clone()
    broken[0, 3] = k.shape[0] + 5
    out, _ = attend(bridge, q, k, v, broken, new, lens)
    assert bridge.error_word(clear=True) == 2
    assert torch.equal(out[new[0]:], good[new[0]:])
    # a length past the table
    out, _ = attend(bridge, q, k, v, table[:, :5], new, lens)
    assert bridge.error_word(clear=True) == 2


@pytest.mark.parametrize("new", [[1, 1], [70, 3]])
def test_attention_nan_reaches_the_rows_that_attend_it_alone(bridge, new):
    lens = [200, 150]
    k, v, table, keys, vals = R.make_cache(lens, 2, 16, 128, BF16, DEV, 65)
    q = torch.randn((sum(new), 16, 128), generator=torch.Generator().manual_seed(66)).to(BF16).to(DEV)
    good, good_lse = attend(bridge, q, k, v, table, new, lens)
    k = k.clone()
    pos = 180 if new[0] > 1 else 77
    k[int(table[0, pos // 16]), 1, pos % 16, 5] = math.nan  # a key of the second key head
    out, lse = attend(bridge, q, k, v, table, new, lens)
    assert bridge.error_word(clear=True) == 0
    first = max(0, pos - (lens[0] - new[0]))  # the first row of sequence 0 that attends it
    assert out[first:new[0], 8:].isnan().all() and lse[first:new[0], 8:].isnan().all()
    assert torch.equal(out[:, :8], good[:, :8]) and torch.equal(out[:first], good[:first])
    assert torch.equal(out[new[0]:], good[new[0]:]) and torch.equal(lse[new[0]:], good_lse[new[0]:])


def values_not_finite(bridge, dtype, heads, kv_heads, d, new, lens, back, value):
    """One element of the value of the key ``back`` places before sequence 0's last one: the rows that attend
    it get it, in its dim alone, and no other row sees it."""

    k, v, table, keys, vals = R.make_cache(lens, kv_heads, 16, d, dtype, DEV, 67)
    q = torch.randn((sum(new), heads, d), generator=torch.Generator().manual_seed(68)).to(dtype)
    pos, dim = lens[0] - 1 - back, d - 3
    v[int(table[0, pos // 16]), kv_heads - 1, pos % 16, dim] = value
    vals[0][kv_heads - 1, pos, dim] = value
    out, lse = attend(bridge, q.to(DEV), k, v, table, new, lens)
    assert bridge.error_word(clear=True) == 0
    scale = 1 / math.sqrt(d)
    ref, ref_lse, mag, reach = R.attention(q, new, lens, keys, vals, scale)
    got, u = out.double().cpu(), R.UNIT[dtype]
    hit = ~torch.isfinite(ref)
    assert hit.any() and not hit[..., :dim].any() and not torch.isfinite(got[hit]).any()
    assert ((got - ref).abs() <= u * ref.abs() + (u + 2.0**-14) * mag)[~hit].all()
    assert ((lse.double().cpu() - ref_lse).abs() <= d * 2.0**-24 * reach + 2.0**-18).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", [
    # dtype, heads, kv_heads, d, new, lengths, back: few rows a key head
    (BF16, 8, 1, 128, [2, 1], [37, 20], 0), (F16, 2, 2, 64, [16], [16], 7), (BF16, 10, 2, 128, [3, 2], [600, 17], 1),
    (F16, 4, 2, 128, [4, 1, 3], [129, 5, 64], 0), (BF16, 5, 5, 64, [9], [9], 8), (F16, 16, 2, 64, [2], [4098], 0),
    (BF16, 6, 3, 128, [8], [33], 3),
])
def test_attention_values_that_are_not_finite_few_rows(bridge, case, value):
    values_not_finite(bridge, *case, value)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", [
    # many rows a key head: blocks of 128 keys, items of 256 rows, pieces cut from a long sequence
    (BF16, 8, 1, 128, [130], [130], 0), (F16, 8, 2, 64, [40, 9], [300, 9], 13), (BF16, 16, 2, 128, [70, 3], [200, 77], 19),
    (F16, 2, 2, 128, [257], [400], 130), (BF16, 10, 2, 128, [50], [4000], 2), (F16, 17, 1, 128, [9], [128], 0),
    (BF16, 40, 1, 64, [30, 50], [30, 51], 28), (BF16, 32, 8, 128, [200, 60, 1], [1000, 60, 500], 140),
])
def test_attention_values_that_are_not_finite_many_rows(bridge, case, value):
    values_not_finite(bridge, *case, value)


def test_attention_no_rows(bridge):
    k, v, table, _, _ = R.make_cache([5], 2, 16, 128, BF16, DEV, 71)
    q = torch.empty((0, 16, 128), dtype=BF16, device=DEV)
    out, _ = attend(bridge, q, k, v, table, [0], [5])
    assert out.shape[0] == 0 and bridge.error_word(clear=True) == 0


@pytest.mark.parametrize("width", [0, 4])
def test_a_batch_of_no_sequences(bridge, width):
    k, v = (torch.zeros((3, 2, 16, 128), dtype=BF16, device=DEV) for _ in range(2))
    q, qkv = torch.empty((0, 16, 128), dtype=BF16, device=DEV), torch.empty((0, 20 * 128), dtype=BF16, device=DEV)
    table, lens = torch.empty((0, width), dtype=torch.int32, device=DEV), torch.empty((0,), dtype=torch.int32, device=DEV)
    start = torch.zeros((1,), dtype=torch.int32, device=DEV)
    ws = bridge.paged_attention_workspace(q, k, table, max_query=0)
    bridge.dispatch_paged_attention(q, k, v, torch.empty_like(q), start, lens, table, ws, max_query=0, stream_ptr=0)
    bridge.dispatch_rope_append_paged(qkv, q, k, v, None, None, start, lens, table, stream_ptr=0)
    torch.cuda.synchronize()
    assert bridge.error_word(clear=True) == 0 and not k.any() and not v.any()


def test_attention_second_tile_idle_for_a_long_time(bridge):
    """Items of one tile first, for longer than 2^17 tries of a barrier last (0.2 s), then items of two: 64
    sequences of 2^27 keys, the same page over and over, for one token of 32 heads, and at the end 300 tokens
    over 400 keys, all in the last worker's share."""

    page, d, n, long = 128, 64, 1 << 27, 64
    g = torch.Generator().manual_seed(83)
    k, v, small, keys, vals = R.make_cache([400], 1, page, d, BF16, DEV, 84)
    table = torch.full((long + 1, n // page), int(small[0, 0]), dtype=torch.int32, device=DEV)
    table[-1, :small.shape[1]] = small[0]
    q = torch.randn((long + 300, 32, d), generator=g).to(BF16).to(DEV)
    out, lse = attend(bridge, q, k, v, table, [1] * long + [300], [n] * long + [400])
    assert bridge.error_word(clear=True) == 0
    check_attention(q[-300:], [300], [400], keys, vals, out[-300:], lse[-300:], 1 / math.sqrt(d))
    # a long sequence attends to 128 keys, to each as often; its 32-bit sums are of that many blocks, and
    # each addition may be off by 2^-23 of the sum
    want, _ = attend(bridge, q[:long], k, v, small[:, :1].repeat(long, 1), [1] * long, [page] * long)
    blocks = long * (n // 128) / (torch.cuda.get_device_properties(0).multi_processor_count - 1)
    bound = (2 * blocks * 2.0**-23 + 2.0**-7) * v[small[0, 0]].abs().max().double()
    assert ((out[:long].double() - want.double()).abs() <= bound).all()


def test_attention_offsets_past_32_bits(bridge):
    """A cache of more than 2^32 elements whose sequences live at its end."""

    page, kh, d = 128, 8, 128
    num = (1 << 32) // (page * kh * d) + 40
    if torch.cuda.mem_get_info()[0] < 2.2 * num * page * kh * d * 2:
        pytest.skip("needs 40 GB of free memory")
    k = torch.empty((num, kh, page, d), dtype=BF16, device=DEV)
    v = torch.empty((num, kh, page, d), dtype=BF16, device=DEV)
    for new, lens in (([1, 1], [700, 300]), ([70, 9], [400, 130])):
        sk, sv, table, keys, vals = R.make_cache(lens, kh, page, d, BF16, DEV, 81)
        at = num - sk.shape[0]
        k[at:], v[at:] = sk, sv
        q = torch.randn((sum(new), 32, d), generator=torch.Generator().manual_seed(82)).to(BF16).to(DEV)
        out, lse = attend(bridge, q, k, v, torch.where(table >= 0, table + at, table), new, lens)
        assert bridge.error_word(clear=True) == 0
        check_attention(q, new, lens, keys, vals, out, lse, 1 / math.sqrt(d))
    del k, v
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ rope + append
def rope_reference(x, cos, sin, interleaved):
    """x [heads, d] in 64 bits rotated by cos/sin [rot / 2]."""

    y = x.clone()
    half = cos.shape[0]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[:, a] = x[:, a] * cos[i] - x[:, b] * sin[i]
        y[:, b] = x[:, b] * cos[i] + x[:, a] * sin[i]
    return y


APPEND = [
    # dtype, q_heads, kv_heads, d, page, rotary, interleaved, bias, new, lengths
    (BF16, 16, 2, 128, 16, 128, False, True, [1], [1]),
    (BF16, 16, 2, 128, 64, 128, False, False, [1, 1, 0, 1], [33, 64, 5, 300]),
    (F16, 5, 5, 64, 32, 32, True, True, [3, 17], [3, 100]),
    (F16, 7, 1, 64, 16, 64, True, False, [40, 1, 5], [57, 2, 90]),
    (BF16, 32, 8, 128, 128, 64, False, True, [130, 3], [131, 257]),
    (BF16, 4, 4, 128, 16, 16, False, False, [9], [20]),
    (BF16, 3, 3, 128, 16, 0, False, True, [9, 2], [20, 2]),  # no rotation
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_rope_append_against_64_bits(bridge, case):
    dtype, qh, kh, d, page, rot, inter, has_bias, new, lens = APPEND[case]
    k, v, table, _, _ = R.make_cache(lens, kh, page, d, dtype, DEV, 300 + case, junk=3.0)
    g = torch.Generator().manual_seed(400 + case)
    rows, heads = sum(new), qh + 2 * kh
    wide = torch.randn((rows, heads * d + 24), generator=g).to(dtype).to(DEV)
    qkv = wide[:, 8:8 + heads * d]  # strided rows
    bias = (0.5 * torch.randn((heads * d,), generator=g)).to(dtype).to(DEV) if has_bias else None
    ang = torch.rand((max(lens) + 2, rot // 2), generator=g, dtype=torch.float64) * 6.28
    cos, sin = ang.cos().float(), ang.sin().float()
    q_out = torch.full((rows, qh, d), 9.0, dtype=dtype, device=DEV)
    start, kv = R.starts(new, DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    before_k, before_v = k.clone(), v.clone()
    bridge.dispatch_rope_append_paged(qkv, q_out, k, v, cos.to(DEV) if rot else None, sin.to(DEV) if rot else None,
                                      start, kv, table, interleaved=inter, bias=bias,
                                      stream_ptr=int(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bridge.error_word(clear=True) == 0
    x = qkv.cpu().double()
    if has_bias:
        x = (x + bias.cpu().double()).float().to(dtype).double()
    x = x.view(rows, heads, d)
    u = R.UNIT[dtype]
    at = 0
    for b, (t, n) in enumerate(zip(new, lens)):
        for i in range(t):
            pos = n - t + i
            turned = rope_reference(x[at, :qh + kh], cos[pos].double(), sin[pos].double(), inter)
            size = rope_reference(x[at, :qh + kh].abs(), torch.ones(rot // 2), -torch.ones(rot // 2), inter).abs()
            bound = u * turned.abs() + 2.0**-22 * (size + x[at, :qh + kh].abs())
            assert ((q_out[at].cpu().double() - turned[:qh]).abs() <= bound[:qh]).all()
            pg, slot = int(table[b, pos // page]), pos % page
            assert ((k[pg, :, slot].cpu().double() - turned[qh:]).abs() <= bound[qh:]).all()
            assert torch.equal(v[pg, :, slot].cpu().double(), x[at, qh + kh:])
            before_k[pg, :, slot] = k[pg, :, slot]
            before_v[pg, :, slot] = v[pg, :, slot]
            at += 1
    # every other slot is as it was
    assert torch.equal(k, before_k) and torch.equal(v, before_v)


def test_rope_append_refuses_positions_and_pages_out_of_range(bridge):
    new, lens = [2, 1, 1, 3], [40, 17, 16, 2]
    k, v, table, _, _ = R.make_cache(lens, 2, 16, 64, BF16, DEV, 91, junk=0.0)
    table[1, 1] = -1            # the page of position 16 is missing
    qkv = torch.randn((7, 8 * 64), device=DEV).to(BF16)
    q_out = torch.full((7, 4, 64), 9.0, dtype=BF16, device=DEV)
    cos = torch.ones((39, 32), device=DEV)  # position 39 has no table row
    sin = torch.zeros((39, 32), device=DEV)
    bridge.dispatch_rope_append_paged(qkv, q_out, k, v, cos, sin, R.starts(new, DEV),
                                      torch.tensor(lens, dtype=torch.int32, device=DEV), table, stream_ptr=0)
    torch.cuda.synchronize()
    assert bridge.error_word(clear=True) == 2
    # written: position 38 of sequence 0, 15 of sequence 2, 0 and 1 of sequence 3
    for row, ok in enumerate([True, False, False, True, False, True, True]):
        assert torch.equal(q_out[row].flatten(), qkv[row, :256]) if ok else (q_out[row] == 9.0).all()


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("layers,pages,shape,moves,tables", [
    (1, 5, (2, 16, 64), 1, False), (3, 40, (2, 16, 128), 17, True), (7, 21, (1, 32, 8), 10, True),
    (2, 9, (3, 128, 128), 4, False), (2, 6, (1, 16, 64), 0, True),
])
def test_kv_pages_copy(bridge, layers, pages, shape, moves, tables):
    g = torch.Generator(device=DEV).manual_seed(pages)
    k = torch.randn((layers, pages, *shape), generator=g, device=DEV).to(F16)
    v = torch.randn((layers, pages, *shape), generator=g, device=DEV).to(F16)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    pairs = torch.stack([order[:moves], order[moves:2 * moves]], 1).contiguous()
    want_k, want_v = k.clone(), v.clone()
    for a, b in pairs.tolist():
        want_k[:, b] = k[:, a]
        want_v[:, b] = v[:, a]
    table = page_map = want = None
    if tables:
        wide = torch.randint(-1, pages, (5, 19), generator=g, device=DEV, dtype=torch.int32)
        wide[0, 3] = pages + 7  # not a page: left alone
        table = wide[:, 2:13]
        page_map = torch.arange(pages, dtype=torch.int32, device=DEV)
        page_map[pairs[:, 0].long()] = pairs[:, 1]
        want = wide.clone()
        for r in range(5):
            for c in range(2, 13):
                e = int(wide[r, c])
                want[r, c] = int(page_map[e]) if 0 <= e < pages else e
    bridge.dispatch_kv_pages_copy(k, v, pairs, block_table=table, page_map=page_map,
                                  stream_ptr=int(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bridge.error_word(clear=True) == 0
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    if tables:
        assert torch.equal(wide, want)


def test_kv_pages_copy_of_one_layer_whose_stride_is_a_page(bridge):
    g = torch.Generator(device=DEV).manual_seed(11)
    k, v = (torch.randn((9, 1, 2, 16, 64), generator=g, device=DEV).to(BF16).transpose(0, 1) for _ in range(2))
    want_k, want_v = k.clone(), v.clone()
    for a, b in ((8, 0), (3, 7)):
        want_k[:, b], want_v[:, b] = k[:, a], v[:, a]
    bridge.dispatch_kv_pages_copy(k, v, torch.tensor([[8, 0], [3, 7]], dtype=torch.int32, device=DEV),
                                  stream_ptr=int(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bridge.error_word(clear=True) == 0 and torch.equal(k, want_k) and torch.equal(v, want_v)


def test_kv_pages_copy_skips_pages_out_of_range(bridge):
    k = torch.randn((2, 6, 1, 16, 64), device=DEV).to(BF16)
    v = k + 1
    want_k, want_v = k.clone(), v.clone()
    want_k[:, 1], want_v[:, 1] = k[:, 4], v[:, 4]
    pairs = torch.tensor([[6, 0], [2, -1], [4, 1]], dtype=torch.int32, device=DEV)
    bridge.dispatch_kv_pages_copy(k, v, pairs, stream_ptr=0)
    torch.cuda.synchronize()
    assert bridge.error_word(clear=True) == 2
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


# ------------------------------------------------------------------ sampling
def sample(bridge, x, u, t=None, k=None, p=None, low=None):
    rows = x.shape[0]

    def col(value, dtype):
        return None if value is None else torch.tensor(value, dtype=dtype, device=DEV)

    tokens = torch.full((rows,), -7, dtype=torch.int32, device=DEV)
    logp = torch.full((rows,), 7.0, device=DEV)
    bridge.dispatch_sample(x, tokens, col(u, torch.float32), temperature=col(t, torch.float32),
                           top_k=col(k, torch.int32), top_p=col(p, torch.float32), min_p=col(low, torch.float32),
                           logprobs=logp, stream_ptr=int(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return tokens.tolist(), logp.tolist()


def check_rows(bridge, x, u, t, k, p, low):
    """Against the definition with the parameters as their 32-bit values."""

    tokens, logp = sample(bridge, x, u, t, k, p, low)
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).double().tolist()  # noqa: E731
    u, t, p, low = f32(u), f32(t), f32(p), f32(low)
    for r in range(x.shape[0]):
        want, want_logp = R.sample_row(x[r].double().tolist(), t[r], k[r], p[r], low[r], u[r])
        assert tokens[r] == want, f"row {r}: {tokens[r]} for {want}"
        assert logp[r] == want_logp or abs(logp[r] - want_logp) <= 2.0**-16


SETTINGS = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.6, 0.0), (0.9, 0, 1.0, 0.2),
            (0.8, 9, 0.8, 0.05), (2.0, 1, 0.5, 0.0), (0.5, 3, 1.0, 1.0), (1.0, 40, 0.999, 0.001), (0.05, 0, 0.9, 0.0),
            (1.0, 0, 0.0, 0.0), (30.0, 0, 0.95, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float32, BF16, F16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 33333])
def test_sample_against_the_definition(bridge, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    rows = len(SETTINGS) * (2 if vocab > 5000 else 4)
    wide = (3.0 * torch.randn((rows, vocab + 5), generator=g)).to(dtype).to(DEV)
    x = wide[:, 3:3 + vocab]  # strided rows at odd offsets
    u = torch.rand((rows,), generator=g).tolist()
    cols = [[SETTINGS[r % len(SETTINGS)][c] for r in range(rows)] for c in range(4)]
    check_rows(bridge, x, u, *cols)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 450001), (BF16, 900003), (F16, 151937)])
def test_sample_long_rows(bridge, dtype, vocab):
    """Rows of several hundred words a thread, odd lengths, every alignment of a row."""

    g = torch.Generator().manual_seed(vocab)
    x = (3.0 * torch.randn((4, vocab), generator=g)).to(dtype).to(DEV)
    u = torch.rand((4,), generator=g).tolist()
    check_rows(bridge, x, u, [0.0, 0.7, 1.0, 0.9], [0, 50, 0, 7], [1.0, 0.9, 0.99, 1.0], [0.0, 0.01, 0.0, 0.1])


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 900001), (BF16, 1700001)])
def test_sample_rows_longer_than_sixteen_blocks_hold(bridge, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    x = (3.0 * torch.randn((3, vocab), generator=g)).to(dtype).to(DEV)
    u = torch.rand((3,), generator=g).tolist()
    check_rows(bridge, x, u, [0.0, 0.7, 0.25], [0, 50, 0], [1.0, 0.9, 0.9], [0.0, 0.01, 0.0])


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_sample_ties_infinities_and_nan(bridge, dtype):
    inf, nan = math.inf, math.nan
    base = [[1.0] * 50, [2.0, 2.0, 1.0, 2.0, 1.0] * 10, [-inf] * 50, [nan] * 50, [-inf] * 49 + [0.5],
            [nan, 1.0, inf, 0.0, inf] * 10, [0.0, -0.0] * 25, [-inf, 3.0, nan, 3.0, 2.0] * 10,
            [torch.finfo(dtype).min] * 50, [torch.finfo(dtype).max, torch.finfo(dtype).min] * 25]
    g = torch.Generator().manual_seed(5)
    rows, us, cols = [], [], [[], [], [], []]
    for row in base:
        for s in SETTINGS:
            rows.append(row)
            us.append(float(torch.rand((1,), generator=g)))
            for c in range(4):
                cols[c].append(s[c])
    check_rows(bridge, torch.tensor(rows, dtype=torch.float64).to(dtype).to(DEV), us, *cols)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 70), (BF16, 5001), (F16, 40000), (BF16, 1700001)])
def test_sample_infinite_temperature(bridge, dtype, vocab):
    """Every entry above -inf is as likely as any other; masked ones and NaN are never drawn."""

    g = torch.Generator().manual_seed(vocab)
    rows = 8 if vocab < 10000 else 4
    x = 3.0 * torch.randn((rows, vocab), generator=g)
    masked = torch.rand((rows, vocab), generator=g) < 0.6
    x = torch.where(masked, -math.inf, x)
    x[1::4, ::7] = math.nan
    x[2::4, 0] = math.inf
    x[3::4, 1:] = -math.inf  # one entry is left
    x[3::4, 0] = 2.0
    u = torch.rand((rows,), generator=g).tolist()
    x = x.to(dtype).to(DEV)
    settings = [(0, 0.5, 0.0), (0, 1.0, 0.0), (9, 1.0, 0.0), (vocab - 1, 0.9, 0.5), (0, 1.0, 1.0)]
    for k, p, low in settings if vocab < 100000 else settings[:1]:
        check_rows(bridge, x, u, [math.inf] * rows, [k] * rows, [p] * rows, [low] * rows)


@pytest.mark.parametrize("dtype", [torch.float32, BF16, F16])
def test_sample_infinite_temperature_and_the_lowest_value(bridge, dtype):
    """A mask of the type's lowest value is finite, so it is as likely as any; min-p of 1 keeps it too."""

    g = torch.Generator().manual_seed(12)
    info = torch.finfo(dtype)
    x = 3.0 * torch.randn((6, 501), generator=g, dtype=torch.float64)
    x = torch.where(torch.rand((6, 501), generator=g) < 0.5, info.min, x)
    x[2::3, ::9] = info.max
    x[1::3, ::5] = -math.inf
    x = x.to(dtype).to(DEV)
    for k, p, low in ((0, 1.0, 0.0), (0, 1.0, 1.0), (0, 0.7, 0.3), (400, 0.9, 1.0)):
        u = torch.rand((6,), generator=g).tolist()
        check_rows(bridge, x, u, [math.inf] * 6, [k] * 6, [p] * 6, [low] * 6)


def test_sample_values_of_every_size(bridge):
    """bf16 values that few entries share, near 0, past 128 and far below, beside ordinary ones."""

    g = torch.Generator().manual_seed(8)
    rows = []
    for r in range(24):
        x = 3.0 * torch.randn((3000,), generator=g)
        if r % 4 == 1:
            x[::3] *= 2.0 ** -torch.randint(5, 20, (1000,), generator=g).float()  # near 0, zeros of both signs
            x[5], x[6] = 0.0, -0.0
            x = x - 2.0 * (x > 1)
        if r % 4 == 2:
            x = x * 40.0
        if r % 4 == 3:
            x = x - 140.0
        rows.append(x)
    x = torch.stack(rows).to(BF16).to(DEV)
    u = torch.rand((24,), generator=g).tolist()
    k = [[0, 7, 0, 2500, 2999, 0][(r // 4) % 6] for r in range(24)]
    p = [[1.0, 0.9, 0.97, 1.0, 0.99, 0.5][(r // 4) % 6] for r in range(24)]
    check_rows(bridge, x, u, [[0.8, 30.0][r % 2] for r in range(24)], k, p, [0.0] * 12 + [1e-4] * 12)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 3000), (BF16, 3000), (F16, 3000), (BF16, 20000)])
def test_sample_many_entries_of_few_values(bridge, dtype, vocab):
    """The kept prefix ends among more entries than fit a list, all of a few values."""

    g = torch.Generator().manual_seed(vocab)
    rows = 24
    x = ((4.0 * 1.5 * torch.randn((rows, vocab), generator=g)).round() / 4.0).to(dtype).to(DEV)
    u = torch.rand((rows,), generator=g).tolist()
    k = [[0, 0, 1500, 2999][r % 4] for r in range(rows)]
    p = [[0.5, 0.9, 0.97, 1.0, 0.99, 0.8][r % 6] for r in range(rows)]
    check_rows(bridge, x, u, [[0.6, 1.0, 3.0][r % 3] for r in range(rows)], k, p, [0.0] * 16 + [1e-3] * 8)


def test_tensors_in_other_memory_are_refused(bridge):
    x = torch.zeros((2, 64), device=DEV)
    tokens, u = torch.zeros((2,), dtype=torch.int32, device=DEV), torch.zeros((2,), device=DEV)
    with pytest.raises(ValueError, match="cuda:0"):
        bridge.dispatch_sample(x, tokens, u.cpu(), stream_ptr=0)
    k = torch.zeros((2, 4, 1, 16, 64), dtype=F16, device=DEV)
    with pytest.raises(ValueError, match="cuda:0"):
        bridge.dispatch_kv_pages_copy(k, k.clone(), torch.zeros((1, 2), dtype=torch.int32), stream_ptr=0)
    start, n, table = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0, 1], [1], [[0]]))
    q, qkv = torch.zeros((1, 1, 64), dtype=F16, device=DEV), torch.zeros((1, 192), dtype=F16, device=DEV)
    ws = bridge.paged_attention_workspace(q, k[0], table, max_query=1)
    with pytest.raises(ValueError, match="cuda:0"):
        bridge.dispatch_paged_attention(q, k[0], k[1], q.clone(), start, n.cpu(), table, ws, max_query=1, stream_ptr=0)
    with pytest.raises(ValueError, match="cuda:0"):
        bridge.dispatch_rope_append_paged(qkv, q, k[0], k[1], None, None, start, n, table.cpu(), stream_ptr=0)


def test_sample_ends_of_the_uniform_range_and_defaults(bridge):
    x = torch.tensor([[0.0, 1.0, -math.inf, 2.0, -math.inf]] * 4, device=DEV)
    tokens, logp = sample(bridge, x, [0.0, 1.0 - 2.0**-24, 0.5, 5.0])
    total = 1 + math.e + math.e**2
    assert tokens == [0, 3, 3, 3]
    assert abs(logp[0] + math.log(total)) < 1e-6 and abs(logp[1] - 2 + math.log(total)) < 1e-6


def test_sample_follows_the_distribution(bridge):
    """Uniform numbers on a fine grid give each token its share to within one step of the grid."""

    n, vocab = 4096, 37
    x = torch.randn((1, vocab), generator=torch.Generator().manual_seed(6)).to(DEV).expand(n, vocab)
    tokens, _ = sample(bridge, x.contiguous(), [(i + 0.5) / n for i in range(n)])
    share = torch.bincount(torch.tensor(tokens), minlength=vocab).double() / n
    assert ((share - torch.softmax(x[0].double().cpu(), 0)).abs() <= 1.01 / n).all()


def test_sample_row_does_not_depend_on_its_batch(bridge):
    g = torch.Generator().manual_seed(7)
    x = (4.0 * torch.randn((130, 50000), generator=g)).to(BF16).to(DEV)
    u = torch.rand((130,), generator=g).tolist()
    cols = [[SETTINGS[r % len(SETTINGS)][c] for r in range(130)] for c in range(4)]
    whole, lw = sample(bridge, x, u, *cols)
    for r in (0, 1, 5, 8, 77, 129):
        one, lo = sample(bridge, x[r:r + 1], u[r:r + 1], *[c[r:r + 1] for c in cols])
        assert one[0] == whole[r] and lo[0] == lw[r]


# ------------------------------------------------------------------ in a captured graph
def captured(work):
    """Runs ``work`` once, captures it, and returns the replay."""

    work()
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        work()

    def replay():
        graph.replay()
        torch.cuda.synchronize()

    return replay


def current():
    return int(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype,rows,vocab", [(BF16, 1, 151936), (BF16, 64, 20000), (torch.float32, 300, 777),
                                              (F16, 3, 40001), (torch.float32, 2, 900001)])
def test_sample_in_a_graph(bridge, dtype, rows, vocab):
    """One block a row, clusters of up to 16 and rows that no cluster holds; every replay on new inputs."""

    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.empty((rows, vocab), dtype=dtype, device=DEV)
    u, temperature, top_p = (torch.empty((rows,), device=DEV) for _ in range(3))
    top_k = torch.empty((rows,), dtype=torch.int32, device=DEV)

    def fill():
        x.copy_(3.0 * torch.randn((rows, vocab), generator=g, device=DEV))
        for t, low, high in ((u, 0.0, 1.0), (temperature, -0.3, 1.5), (top_p, 0.5, 1.1)):
            t.copy_(low + (high - low) * torch.rand((rows,), generator=g, device=DEV))
        top_k.copy_(torch.randint(0, 60, (rows,), generator=g, device=DEV))

    def into(tokens, logp):
        bridge.dispatch_sample(x, tokens, u, temperature=temperature, top_k=top_k, top_p=top_p, logprobs=logp,
                               stream_ptr=current())

    fill()
    tokens, logp = torch.zeros((rows,), dtype=torch.int32, device=DEV), torch.zeros((rows,), device=DEV)
    want, want_logp = torch.zeros_like(tokens), torch.zeros_like(logp)
    replay = captured(lambda: into(tokens, logp))
    for _ in range(3):
        fill()
        replay()
        into(want, want_logp)
        torch.cuda.synchronize()
        assert torch.equal(tokens, want) and torch.equal(logp, want_logp)


@pytest.mark.parametrize("new", [[1, 1, 1], [700, 1, 30]])
def test_rope_append_in_a_graph(bridge, new):
    """The lengths are device data: a replay appends where they say."""

    lens = [800, 40, 90]
    k, v, table, _, _ = R.make_cache([n + 20 for n in lens], 2, 16, 128, BF16, DEV, 97, junk=0.0)
    start, kv = R.starts(new, DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    qkv = torch.randn((sum(new), 20 * 128), generator=torch.Generator(device=DEV).manual_seed(98), device=DEV).to(BF16)
    ang = torch.rand((900, 64), generator=torch.Generator(device=DEV).manual_seed(99), device=DEV) * 6.28
    cos, sin = ang.cos(), ang.sin()
    q = torch.zeros((sum(new), 16, 128), dtype=BF16, device=DEV)

    def into(q, k, v):
        bridge.dispatch_rope_append_paged(qkv, q, k, v, cos, sin, start, kv, table, stream_ptr=current())

    replay = captured(lambda: into(q, k, v))
    for step in range(3):
        kv.add_(step + 1)
        qkv.mul_(0.5)
        want_q, want_k, want_v = q.clone(), k.clone(), v.clone()
        into(want_q, want_k, want_v)
        replay()
        assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(v, want_v)
    assert bridge.error_word(clear=True) == 0


def test_kv_pages_copy_in_a_graph(bridge):
    g = torch.Generator(device=DEV).manual_seed(21)
    k, v = (torch.randn((3, 12, 2, 16, 64), generator=g, device=DEV).to(BF16) for _ in range(2))
    pairs = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    table = torch.randint(-1, 12, (3, 5), generator=g, device=DEV, dtype=torch.int32)
    page_map = torch.arange(12, dtype=torch.int32, device=DEV)

    def into(k, v, table):
        bridge.dispatch_kv_pages_copy(k, v, pairs, block_table=table, page_map=page_map, stream_ptr=current())

    replay = captured(lambda: into(k, v, table))
    for new in ([[4, 5], [6, 0]], [[11, 2], [8, 9]]):
        pairs.copy_(torch.tensor(new, dtype=torch.int32))
        page_map.copy_(torch.arange(12, dtype=torch.int32))
        for a, b in new:
            page_map[a] = b
        want = k.clone(), v.clone(), table.clone()
        into(*want)
        replay()
        assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and torch.equal(table, want[2])
        assert torch.equal(k[:, new[0][1]], k[:, new[0][0]])
    assert bridge.error_word(clear=True) == 0


# ------------------------------------------------------------------ refusals of the C entries
def test_native_refusals(bridge):
    from kudacuda_b200.kudacuda_sidecar import NativeCudaError

    k, v, table, _, _ = R.make_cache([40], 2, 16, 128, BF16, DEV, 95)
    start, kv = R.starts([1], DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    q = torch.zeros((1, 16, 128), dtype=BF16, device=DEV)
    out = torch.empty_like(q)
    ws = bridge.paged_attention_workspace(q, k, table, max_query=1)

    def attention(**kw):
        a = dict(q=q, k=k, v=v, out=out, start=start, kv=kv, table=table, ws=ws, max_query=1, scale=None) | kw
        bridge.dispatch_paged_attention(a["q"], a["k"], a["v"], a["out"], a["start"], a["kv"], a["table"], a["ws"],
                                        max_query=a["max_query"], scale=a["scale"], stream_ptr=0)

    def pages(shape):
        return dict(k=torch.zeros(shape, dtype=BF16, device=DEV), v=torch.zeros(shape, dtype=BF16, device=DEV))

    with pytest.raises(NativeCudaError, match="page_size"):
        attention(**pages((4, 2, 24, 128)))
    with pytest.raises(NativeCudaError, match="head_dim"):
        attention(q=torch.zeros((1, 16, 96), dtype=BF16, device=DEV),
                  out=torch.zeros((1, 16, 96), dtype=BF16, device=DEV), **pages((4, 2, 16, 96)))
    with pytest.raises(NativeCudaError, match="multiple of kv_heads"):
        attention(**pages((4, 3, 16, 128)))
    with pytest.raises(NativeCudaError, match="max_query"):
        attention(max_query=2)
    with pytest.raises(NativeCudaError, match="scale"):
        attention(scale=-1.0)
    with pytest.raises(NativeCudaError, match="aligned"):
        attention(q=torch.zeros((2049,), dtype=BF16, device=DEV)[1:].view(1, 16, 128))
    x = torch.zeros((2, 10), device=DEV)
    with pytest.raises(NativeCudaError, match="page_bytes"):
        bridge.dispatch_kv_pages_copy(torch.zeros((1, 4, 3), dtype=BF16, device=DEV),
                                      torch.zeros((1, 4, 3), dtype=BF16, device=DEV),
                                      torch.zeros((1, 2), dtype=torch.int32, device=DEV), stream_ptr=0)
    with pytest.raises(NativeCudaError, match="rotary_dim"):
        bridge.dispatch_rope_append_paged(torch.zeros((1, 20 * 128), dtype=BF16, device=DEV), out, k, v,
                                          torch.zeros((64, 20), device=DEV), torch.zeros((64, 20), device=DEV), start,
                                          kv, table, stream_ptr=0)
    with pytest.raises(NativeCudaError, match="vocab"):
        bridge.dispatch_sample(torch.empty((2, 0), device=DEV), torch.zeros((2,), dtype=torch.int32, device=DEV),
                               x[:, 0].contiguous(), stream_ptr=0)
    torch.cuda.synchronize()
    assert bridge.error_word(clear=True) == 0


@pytest.mark.parametrize("kw,word", [(dict(num_pages=1 << 60), "num_pages"), (dict(num_pages=(1 << 59) + 1), "num_pages"),
                                     (dict(width=1 << 60), "table_width"), (dict(width=(1 << 60) + 1), "table_width")])
def test_native_refuses_sizes_whose_products_wrap(bridge, kw, word):
    k, v, table, _, _ = R.make_cache([40], 2, 16, 128, BF16, DEV, 95)
    start, kv = R.starts([1], DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    q = torch.zeros((1, 16, 128), dtype=BF16, device=DEV)
    out, ws = torch.empty_like(q), bridge.paged_attention_workspace(q, k, table, max_query=1)
    width, pages = kw.get("width", table.shape[1]), kw.get("num_pages", k.shape[0])
    rc = bridge.lib.kudacuda_sm100_paged_attention(
        bridge.engine_handle, 2, q.data_ptr(), 2048, k.data_ptr(), v.data_ptr(), out.data_ptr(), 2048, 0, ws.data_ptr(),
        ws.nbytes, start.data_ptr(), kv.data_ptr(), table.data_ptr(), width, width, 1, 1, 1, 16, 2, 128, pages, 16, 0.1, 0)
    assert rc == 1 and word in bridge.lib.kudacuda_last_error(bridge.engine_handle).decode()
