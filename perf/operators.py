"""What is measured of the paged-cache serving operators: rotary positions with
the append into a paged KV cache, attention of new tokens over that cache,
page copies, and sampling.

Every operator has a plain form (elementary torch operations in 32 bits, one
rounding at the end) beside the framework's own call; ``own`` selects.  A
ragged batch is described the same way everywhere: ``query_start`` (int32
[B + 1], cumulative rows), ``kv_len`` (int32 [B], each sequence's length with
its new tokens) and ``block_table`` (int32 [B, n], page numbers, -1 where a
sequence has none); pages are [num_pages, kv_heads, page_size, head_dim].
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# sampling works on whole-number masses of this scale, so sums do not depend on their order
MASS_ONE = float(2**38)

_BRIDGE = None


def _bridge():
    """The process's handle of the library, as a program keeps one."""

    global _BRIDGE
    if _BRIDGE is None:
        from kudacuda_b200.kudacuda_sidecar import KudaCudaBridge

        _BRIDGE = KudaCudaBridge(device_id=0)
    return _BRIDGE


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one user's next token in a short conversation: latency alone
        {"name": "attention_decode_one", "op": "attention", "batch": 1, "new_min": 1, "new_max": 1, "kv_min": 509,
         "kv_max": 509, "q_heads": 16, "kv_heads": 2, "head_dim": 128, "page": 16, "dtype": "bf16", "shape": 1},
        # a full decode batch of the batched configuration, ragged lengths to 2048
        {"name": "attention_decode_batch", "op": "attention", "batch": 64, "new_min": 1, "new_max": 1, "kv_min": 32,
         "kv_max": 2048, "q_heads": 16, "kv_heads": 2, "head_dim": 128, "page": 64, "dtype": "bf16", "shape": 2},
        # two long documents being answered: the cache read is everything
        {"name": "attention_decode_long", "op": "attention", "batch": 2, "new_min": 1, "new_max": 1, "kv_min": 70001,
         "kv_max": 130001, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "dtype": "f16", "shape": 3},
        # a serving step that mixes decoding sequences with pieces of prompts
        {"name": "attention_mixed", "op": "attention", "batch": 24, "new_min": 1, "new_max": 77, "kv_min": 100,
         "kv_max": 4096, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "dtype": "bf16", "shape": 4},
        # prompts in chunks of 2048 tokens over what is already cached
        {"name": "attention_chunk_large", "op": "attention", "batch": 4, "new_min": 2048, "new_max": 2048,
         "kv_min": 8192, "kv_max": 8192, "q_heads": 16, "kv_heads": 2, "head_dim": 128, "page": 64, "dtype": "bf16",
         "shape": 5},
        # one decode step of 64 sequences: a row each, into 64 places
        {"name": "append_decode_batch", "op": "append", "batch": 64, "new_min": 1, "new_max": 1, "kv_min": 32,
         "kv_max": 2048, "q_heads": 16, "kv_heads": 2, "head_dim": 128, "page": 64, "rotary": 128,
         "interleaved": False, "bias": True, "dtype": "bf16", "shape": 6},
        # prompts of 8192 tokens in all, interleaved pairs on half of the head
        {"name": "append_chunk_large", "op": "append", "batch": 5, "new_min": 1100, "new_max": 2100, "kv_min": 2100,
         "kv_max": 8000, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "rotary": 64,
         "interleaved": True, "bias": False, "dtype": "f16", "shape": 7},
        # a request forked into eight answers: the part-filled last page of each is copied, all layers
        {"name": "pages_fork", "op": "pages", "layers": 36, "pages": 96, "moves": 8, "tables": 0, "table_width": 0,
         "kv_heads": 2, "page": 64, "head_dim": 128, "dtype": "bf16", "shape": 8},
        # a cache compacted after half of its sequences left, tables rewritten
        {"name": "pages_compact", "op": "pages", "layers": 32, "pages": 700, "moves": 300, "tables": 24,
         "table_width": 64, "kv_heads": 8, "page": 16, "head_dim": 128, "dtype": "f16", "shape": 9},
        # one user's next token out of the full vocabulary
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 151936, "dtype": "bf16", "shape": 10},
        # a batch of users, each with settings of their own
        {"name": "sample_batch", "op": "sample", "rows": 64, "vocab": 151936, "dtype": "bf16", "shape": 11},
        # many short-vocabulary rows in 32 bits, an odd width
        {"name": "sample_many", "op": "sample", "rows": 333, "vocab": 50257, "dtype": "f32", "shape": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "append", "pages", "sample"))
    case = {"op": op, "shape": rng.randrange(1 << 30)}
    if op in ("attention", "append"):
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        case |= {"kv_heads": kv_heads, "q_heads": kv_heads * rng.choice((1, 2, 4, 5, 7, 8)),
                 "head_dim": rng.choice((64, 128, 128)), "page": rng.choice((16, 32, 64, 128)),
                 "dtype": rng.choice(("bf16", "bf16", "f16"))}
    if op == "attention":
        case["batch"] = _log_int(rng, 1, 64)
        new = rng.choice((1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 2048)))
        # no more work than the largest listed case: products (and the plain form's score matrix), bytes of the cache
        case["new_max"] = new = min(new, int(math.sqrt(5.0e8 / (case["batch"] * case["q_heads"]))))
        case["new_min"] = rng.randint(1, new)
        cap = min(131072.0, 8.0e8 / (case["batch"] * kv_heads * case["head_dim"] * 4),
                  5.0e8 / (case["batch"] * case["q_heads"] * new))
        case["kv_max"] = max(case["new_max"], _log_int(rng, 16, max(17.0, cap)))
        case["kv_min"] = max(case["new_max"], _log_int(rng, max(1, case["kv_max"] // 16), case["kv_max"]))
    elif op == "append":
        case["batch"] = _log_int(rng, 1, 64)
        case["new_max"] = _log_int(rng, 1, max(2, 8000 // case["batch"]))
        case["new_min"] = rng.randint(1, case["new_max"])
        case["kv_min"] = case["new_max"]
        case["kv_max"] = max(case["new_max"], min(_log_int(rng, 16, 8192), 65536 // case["batch"]))
        case["rotary"] = rng.choice((case["head_dim"], case["head_dim"] // 2, 32))
        case["interleaved"] = rng.random() < 0.5
        case["bias"] = rng.random() < 0.5
    elif op == "pages":
        case |= {"layers": rng.choice((1, 7, 24, 32, 36)), "moves": _log_int(rng, 1, 300),
                 "kv_heads": rng.choice((1, 2, 4, 8)), "page": rng.choice((16, 32)),
                 "head_dim": rng.choice((64, 128)), "dtype": rng.choice(("bf16", "f16")),
                 "tables": rng.choice((0, 1, 17, 64)), "table_width": rng.choice((9, 64, 129))}
        one = 8 * case["layers"] * case["kv_heads"] * case["page"] * case["head_dim"]
        case["moves"] = min(case["moves"], int(1.2e9 / one))
        case["pages"] = 2 * case["moves"] + rng.randint(1, 64)
    else:
        case |= {"rows": _log_int(rng, 1, 333), "dtype": rng.choice(("bf16", "f16", "f32"))}
        case["vocab"] = min(_log_int(rng, 1000, 160000), 16_000_000 // case["rows"])
    return case


def _lengths(case):
    """(new tokens, cached length with them) of every sequence of a ragged case."""

    r = random.Random(case["shape"])
    new = [r.randint(case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    return new, [max(n, _log_int(r, case["kv_min"], case["kv_max"])) for n in new]


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) * 7919 + 13)


def _cache(case, kv, g, fill):
    """Pages in shuffled order, tables with -1 where a sequence has no page."""

    page, d = case["page"], case["head_dim"]
    need = [(n + page - 1) // page for n in kv]
    num = sum(need) + 3
    shape = (num, case["kv_heads"], page, d)
    dtype = TYPES[case["dtype"]]
    if fill:
        # keys carry a few strong channels, as rotated keys do
        gain = 0.6 + 1.4 * torch.rand((d,), generator=g, device=DEVICE) ** 4
        k = (torch.randn(shape, generator=g, device=DEVICE) * gain).to(dtype)
        v = torch.randn(shape, generator=g, device=DEVICE).to(dtype)
    else:
        k, v = torch.zeros(shape, dtype=dtype, device=DEVICE), torch.zeros(shape, dtype=dtype, device=DEVICE)
    order = torch.randperm(num, generator=g, device=DEVICE)[: sum(need)].to(torch.int32)
    width = max(need)
    counts = torch.tensor(need, device=DEVICE)
    held = torch.arange(width, device=DEVICE)[None] < counts[:, None]
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device=DEVICE)
    table[held] = order
    return k, v, table


def _ragged(new, kv):
    start = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEVICE)
    return start, torch.tensor(kv, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    state = {"case": case}
    if op in ("attention", "append"):
        new, kv = _lengths(case)
        qh, kh, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        dtype = TYPES[case["dtype"]]
        rows = sum(new)
        state["start"], state["kv_len"] = _ragged(new, kv)
        state["k"], state["v"], state["table"] = _cache(case, kv, g, op == "attention")
        state["max_new"] = max(new)
        if op == "attention":
            state["q"] = (1.3 * torch.randn((rows, qh, d), generator=g, device=DEVICE)).to(dtype)
            state["out"] = torch.empty((rows, qh, d), dtype=dtype, device=DEVICE)
            state["lse"] = torch.empty((rows, qh), dtype=torch.float32, device=DEVICE)
        else:
            rot = case["rotary"]
            state["qkv"] = torch.randn((rows, (qh + 2 * kh) * d), generator=g, device=DEVICE).to(dtype)
            state["bias"] = (0.02 * torch.randn(((qh + 2 * kh) * d,), generator=g, device=DEVICE)).to(dtype) \
                if case["bias"] else None
            inv = 1.0e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
            ang = torch.arange(max(kv), dtype=torch.float64, device=DEVICE)[:, None] * inv
            state["cos"], state["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
            state["q_out"] = torch.empty((rows, qh, d), dtype=dtype, device=DEVICE)
    elif op == "pages":
        shape = (case["layers"], case["pages"], case["kv_heads"], case["page"], case["head_dim"])
        dtype = TYPES[case["dtype"]]
        state["k"] = torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)
        state["v"] = torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)
        order = torch.randperm(case["pages"], generator=g, device=DEVICE).to(torch.int32)
        n = case["moves"]
        state["pairs"] = torch.stack([order[:n], order[n: 2 * n]], dim=1).contiguous()
        state["table"] = state["map"] = None
        if case["tables"]:
            to = torch.arange(case["pages"], dtype=torch.int32, device=DEVICE)
            to[order[:n].long()] = order[n: 2 * n]
            state["map"] = to
            # tables name pages that move and pages that stay; unused entries are -1
            held = torch.cat([order[:n], order[2 * n:]]).long()
            pick = torch.randint(0, held.numel(), (case["tables"], case["table_width"]), generator=g, device=DEVICE)
            table = held[pick].to(torch.int32)
            blank = torch.rand(table.shape, generator=g, device=DEVICE) < 0.2
            state["table"] = table.masked_fill(blank, -1)
    else:
        rows, vocab = case["rows"], case["vocab"]
        # a few likely tokens over a long tail, at shuffled places
        rank = torch.argsort(torch.rand((rows, vocab), generator=g, device=DEVICE), dim=1).float() + 1.0
        steep = 1.0 + 0.8 * torch.rand((rows, 1), generator=g, device=DEVICE)
        logits = 12.0 - steep * rank.log() + 0.3 * torch.randn((rows, vocab), generator=g, device=DEVICE)
        state["logits"] = logits.to(TYPES[case["dtype"]])
        # settings of real requests: greedy, temperature alone, top-k, top-p, min-p, and all together
        kind = (torch.arange(rows, device=DEVICE) + 5) % 6
        state["temperature"] = torch.where(kind == 0, 0.0, 0.6 + 0.6 * torch.rand((rows,), generator=g, device=DEVICE))
        k = torch.randint(1, 101, (rows,), generator=g, device=DEVICE, dtype=torch.int32)
        state["top_k"] = torch.where((kind == 2) | (kind == 5), k, torch.zeros_like(k))
        p = 0.8 + 0.19 * torch.rand((rows,), generator=g, device=DEVICE)
        state["top_p"] = torch.where((kind == 3) | (kind == 5), p, torch.ones_like(p))
        low = 0.02 + 0.08 * torch.rand((rows,), generator=g, device=DEVICE)
        state["min_p"] = torch.where((kind == 4) | (kind == 5), low, torch.zeros_like(low))
        state["uniform"] = torch.rand((rows,), generator=g, device=DEVICE)
        state["tokens"] = torch.empty((rows,), dtype=torch.int32, device=DEVICE)
        state["logprobs"] = torch.empty((rows,), dtype=torch.float32, device=DEVICE)
    return state


# ------------------------------------------------------------------ plain forms
def _places(state, rows):
    """Sequence, index within it and position of every new row."""

    start = state["start"].long()
    r = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(start[1:], r, right=True)
    i = r - start[seq]
    pos = state["kv_len"].long()[seq] - (start[seq + 1] - start[seq]) + i
    return seq, i, pos


def _pages_of(pages, table):
    """Every sequence's keys or values in order: [B, kv_heads, n * page, d] in 32 bits."""

    b, n = table.shape
    x = pages[table.clamp(min=0).long()].float()
    return x.permute(0, 2, 1, 3, 4).reshape(b, x.shape[2], n * x.shape[3], x.shape[4])


def _plain_attention(state):
    q = state["q"]
    rows, qh, d = q.shape
    k, v = _pages_of(state["k"], state["table"]), _pages_of(state["v"], state["table"])
    b, kh, length, _ = k.shape
    most, group = state["max_new"], qh // kh
    seq, i, pos = _places(state, rows)
    padded = torch.zeros((b, most, qh, d), device=DEVICE)
    padded[seq, i] = q.float()
    last = torch.full((b, most), -1, dtype=torch.long, device=DEVICE)
    last[seq, i] = pos
    qq = padded.view(b, most, kh, group, d).permute(0, 2, 3, 1, 4).reshape(b, kh, group * most, d)
    s = (qq @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(b, kh, group, most, length)
    s.masked_fill_((torch.arange(length, device=DEVICE) > last[:, :, None])[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-1.0e30)
    p = s.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    o = (p.view(b, kh, group * most, length) @ v).view(b, kh, group, most, d) / z.clamp(min=1.0e-30)
    lse = (m + z.log()).squeeze(-1)
    out = o.permute(0, 3, 1, 2, 4).reshape(b, most, qh, d)[seq, i]
    return {"out": out.to(q.dtype), "lse": lse.permute(0, 3, 1, 2).reshape(b, most, qh)[seq, i]}


def _plain_append(state):
    case = state["case"]
    qh, kh, d, rot = case["q_heads"], case["kv_heads"], case["head_dim"], case["rotary"]
    dtype = state["qkv"].dtype
    rows = state["qkv"].shape[0]
    x = state["qkv"].float()
    if state["bias"] is not None:
        x = (x + state["bias"].float()).to(dtype).float()
    x = x.view(rows, qh + 2 * kh, d)
    seq, _, pos = _places(state, rows)
    c, s = state["cos"][pos][:, None], state["sin"][pos][:, None]
    turned = x[:, : qh + kh].clone()
    if case["interleaved"]:
        x0, x1 = x[:, : qh + kh, 0:rot:2], x[:, : qh + kh, 1:rot:2]
        turned[..., 0:rot:2], turned[..., 1:rot:2] = x0 * c - x1 * s, x1 * c + x0 * s
    else:
        x0, x1 = x[:, : qh + kh, : rot // 2], x[:, : qh + kh, rot // 2: rot]
        turned[..., : rot // 2], turned[..., rot // 2: rot] = x0 * c - x1 * s, x1 * c + x0 * s
    page = state["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    state["k"][page, :, slot] = turned[:, qh:].to(dtype)
    state["v"][page, :, slot] = x[:, qh + kh:].to(dtype)
    return {"q": turned[:, :qh].to(dtype), "k": state["k"], "v": state["v"]}


def _plain_pages(state):
    src, dst = state["pairs"][:, 0].long(), state["pairs"][:, 1].long()
    state["k"][:, dst] = state["k"][:, src]
    state["v"][:, dst] = state["v"][:, src]
    got = {"k": state["k"], "v": state["v"]}
    if state["table"] is not None:
        table = state["table"]
        got["table"] = torch.where(table >= 0, state["map"][table.clamp(min=0).long()], table)
    return got


def _plain_sample(state):
    x = state["logits"].float()
    rows, vocab = x.shape
    x = torch.where(x.isnan(), -math.inf, x)
    m, first = x.max(dim=1, keepdim=True)
    t = state["temperature"][:, None]
    inv = 1.0 / torch.where(t > 0, t, torch.ones_like(t))
    w = torch.where(x == m, 1.0, torch.exp((x - m) * inv))
    mass = torch.round(w * MASS_ONE).to(torch.int64)
    # in order of value, the lowest index first among equals
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    ordered = mass.gather(1, order)
    place = torch.arange(vocab, device=DEVICE)[None]
    k = state["top_k"][:, None]
    within_k = (place < k) | (k <= 0)
    before = ordered.cumsum(1) - ordered
    total = (ordered * within_k).sum(1, keepdim=True)
    p = state["top_p"][:, None]
    reach = (p.double() * total.double()).ceil().to(torch.int64).clamp(min=1)
    within_p = (before < reach) | ~(p < 1)
    keep = torch.zeros_like(within_k).scatter(1, order, within_k & within_p)
    keep &= ~(w < state["min_p"][:, None].clamp(max=1.0))
    kept = mass * keep
    cum = kept.cumsum(1)
    whole = cum[:, -1:]
    aim = (state["uniform"][:, None].double() * whole.double()).floor().to(torch.int64)
    aim = aim.clamp(min=0).minimum(whole - 1)
    token = (cum <= aim).sum(1, keepdim=True)
    logprob = (mass.gather(1, token).double() / whole.double()).log().float()
    # the lowest index of the largest value where the temperature is 0
    lowest = torch.where(x == m, place, vocab).amin(1, keepdim=True)
    greedy = ~(t > 0)
    token = torch.where(greedy, lowest, token)
    logprob = torch.where(greedy, 0.0, logprob)
    none = m == -math.inf
    return {"tokens": torch.where(none, -1, token).squeeze(1).to(torch.int32),
            "logprobs": torch.where(none, -math.inf, logprob).squeeze(1)}


# ------------------------------------------------------------------ the framework's calls
def _own_attention(state):
    br = _bridge()
    if "workspace" not in state:
        state["workspace"] = br.paged_attention_workspace(
            state["q"], state["k"], state["table"], max_query=state["max_new"])
    br.dispatch_paged_attention(state["q"], state["k"], state["v"], state["out"], state["start"], state["kv_len"],
                                state["table"], state["workspace"], max_query=state["max_new"], lse=state["lse"],
                                stream_ptr=torch.cuda.current_stream().cuda_stream)
    return {"out": state["out"], "lse": state["lse"]}


def _own_append(state):
    case = state["case"]
    _bridge().dispatch_rope_append_paged(
        state["qkv"], state["q_out"], state["k"], state["v"], state["cos"], state["sin"], state["start"],
        state["kv_len"], state["table"], interleaved=case["interleaved"], bias=state["bias"],
        stream_ptr=torch.cuda.current_stream().cuda_stream)
    return {"q": state["q_out"], "k": state["k"], "v": state["v"]}


def _own_pages(state):
    _bridge().dispatch_kv_pages_copy(state["k"], state["v"], state["pairs"], block_table=state["table"],
                                     page_map=state["map"], stream_ptr=torch.cuda.current_stream().cuda_stream)
    got = {"k": state["k"], "v": state["v"]}
    if state["table"] is not None:
        got["table"] = state["table"]
    return got


def _own_sample(state):
    _bridge().dispatch_sample(state["logits"], state["tokens"], state["uniform"], temperature=state["temperature"],
                              top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"],
                              logprobs=state["logprobs"], stream_ptr=torch.cuda.current_stream().cuda_stream)
    return {"tokens": state["tokens"], "logprobs": state["logprobs"]}


PLAIN = {"attention": _plain_attention, "append": _plain_append, "pages": _plain_pages, "sample": _plain_sample}
OWN = {"attention": _own_attention, "append": _own_append, "pages": _own_pages, "sample": _own_sample}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "f32" else 2
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + 28 * case["rows"], "flops": 4 * n}
    if op == "pages":
        one = case["kv_heads"] * case["page"] * case["head_dim"] * size
        return {"bytes": 4 * case["layers"] * case["moves"] * one + 8 * case["moves"]
                + 8 * case["tables"] * case["table_width"], "flops": 0}
    new, kv = _lengths(case)
    qh, kh, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    if op == "attention":
        keys = sum(sum(range(n - t + 1, n + 1)) for t, n in zip(new, kv))
        return {"bytes": sum(new) * qh * (2 * d * size + 4) + 2 * sum(kv) * kh * d * size
                + 4 * sum((n + page - 1) // page for n in kv) + 8 * len(kv),
                "flops": 4 * d * qh * keys}
    rot = case["rotary"]
    spans = sorted((n - t, n) for t, n in zip(new, kv))
    places, end = 0, 0
    for lo, hi in spans:
        places += max(0, hi - max(lo, end))
        end = max(end, hi)
    return {"bytes": 2 * sum(new) * (qh + 2 * kh) * d * size + places * rot * 4
            + ((qh + 2 * kh) * d * size if case["bias"] else 0),
            "flops": 3 * sum(new) * (qh + kh) * rot}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "pages": _exact_pages,
            "sample": _exact_sample}[case["op"]](case, state)


def _exact_attention(case, state):
    new, kv = _lengths(case)
    kh, d, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["q_heads"] // kh
    q = state["q"].double()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device=DEVICE)
    at = 0
    for b, (t, n) in enumerate(zip(new, kv)):
        ids = state["table"][b, : (n + page - 1) // page].long()
        for h in range(kh):
            keys = state["k"][ids, h].reshape(-1, d)[:n].double()
            vals = state["v"][ids, h].reshape(-1, d)[:n].double()
            for g in range(group):
                for r in range(0, t, 512):
                    e = min(t, r + 512)
                    x = (q[at + r: at + e, h * group + g] / math.sqrt(d)) @ keys.T
                    allowed = torch.arange(n, device=DEVICE)[None] \
                        <= (n - t + torch.arange(r, e, device=DEVICE))[:, None]
                    x = x.masked_fill(~allowed, -math.inf)
                    lse[at + r: at + e, h * group + g] = torch.logsumexp(x, dim=1)
                    out[at + r: at + e, h * group + g] = torch.softmax(x, dim=1) @ vals
        at += t
    return {"out": out, "lse": lse}


def _exact_append(case, state):
    new, kv = _lengths(case)
    qh, kh, d, rot, page = (case[x] for x in ("q_heads", "kv_heads", "head_dim", "rotary", "page"))
    x = state["qkv"].double()
    if state["bias"] is not None:
        x = (x + state["bias"].double()).to(state["qkv"].dtype).double()
    x = x.view(-1, qh + 2 * kh, d)
    k, v = state["k"].double(), state["v"].double()
    qs, at = [], 0
    for b, (t, n) in enumerate(zip(new, kv)):
        pos = torch.arange(n - t, n, device=DEVICE)
        rows = x[at: at + t]
        z = torch.complex(state["cos"][pos].double(), state["sin"][pos].double())[:, None]
        head = rows[:, : qh + kh, :rot]
        pair = head.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else \
            head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
        turned = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
        full = torch.cat([turned, rows[:, : qh + kh, rot:]], dim=-1)
        qs.append(full[:, :qh])
        ids = state["table"][b].long()[pos // page]
        k[ids, :, pos % page] = full[:, qh:]
        v[ids, :, pos % page] = rows[:, qh + kh:]
        at += t
    return {"q": torch.cat(qs), "k": k, "v": v}


def _exact_pages(case, state):
    pairs = state["pairs"].tolist()
    out = {}
    for name in ("k", "v"):
        x = state[name].double()
        for src, dst in pairs:
            x[:, dst] = x[:, src]
        out[name] = x
    if state["table"] is not None:
        to = dict(pairs)
        rows = [[to.get(e, e) for e in row] for row in state["table"].tolist()]
        out["table"] = torch.tensor(rows, dtype=torch.int32, device=DEVICE)
    return out


def _exact_sample(case, state):
    logprobs = []
    for r in range(case["rows"]):
        x = state["logits"][r].double()
        t, k, p, low, u = (float(state[s][r]) for s in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        if t <= 0:
            logprobs.append(0.0)
            continue
        w = torch.exp((x - x.max()) / t)
        value, order = torch.sort(w, descending=True, stable=True)
        count = int(k) if k > 0 else case["vocab"]
        if p < 1:
            run_ = value[:count].cumsum(0)
            count = min(count, int((run_ < p * run_[-1]).sum()) + 1)
        kept, _ = torch.sort(order[:count])
        kept = kept[w[kept] >= low]
        run_ = w[kept].cumsum(0)
        hit = kept[min(int((run_ <= u * run_[-1]).sum()), kept.numel() - 1)]
        logprobs.append(float(torch.log(w[hit] / run_[-1])))
    return {"tokens": None, "logprobs": torch.tensor(logprobs, dtype=torch.float64, device=DEVICE)}
