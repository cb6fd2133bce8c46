"""Several continuations of one prompt, as a list of cases that can be timed and checked.

Three operators that a step of such work is made of:

``attention``  single tokens of sequences that share their first keys in groups: a request's beams or samples, or users of one
               system prompt.  The shared keys lie in the same pages of the cache.
``select``     the best continuations of every request over its beams and the vocabulary.
``reorder``    every beam takes over what its parent held behind the shared keys: rows of states, or pages.

A case's keys.  ``attention``: ``groups`` of up to ``beams`` sequences (``ragged``: from 1 to ``beams``), ``shared`` keys (``ragged``:
from half of it up), up to ``own`` keys of a sequence's own; ``heads``, ``kv_heads``, ``head_dim``, ``dtype``, ``page``, ``sinks``.
``select``: ``requests``, ``beams``, ``vocab``, ``keep``, ``masked`` (one token in so many is forbidden; 0: none), ``first`` (a
request's first step: one beam alone has begun).  ``reorder``: ``requests``, ``beams``, ``rows`` per beam, ``layers`` of
``width`` elements a row, ``dtype``; the layers' rows lie in one tensor, as a page group's do.
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False
DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def attention(name, groups, beams, shared, own_keys, heads, kv_heads, head_dim=128, dtype="bfloat16", page=16, ragged=False, sinks=False):
    return dict(name=name, op="attention", groups=groups, beams=beams, shared=shared, own=own_keys, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                page=page, ragged=ragged, sinks=sinks)


def select(name, requests, beams, vocab, keep, masked=0, first=False):
    return dict(name=name, op="select", requests=requests, beams=beams, vocab=vocab, keep=keep, masked=masked, first=first)


def reorder(name, requests, beams, rows, layers, width, dtype):
    return dict(name=name, op="reorder", requests=requests, beams=beams, rows=rows, layers=layers, width=width, dtype=dtype)


def listed():
    return [
        # one request's four beams a few tokens behind a short prompt: the launch and the latency of one pass decide
        attention("attention 1x4 short", 1, 4, 301, 24, 12, 2),
        # eight requests with four beams each, prompts of unequal length
        attention("attention 8x4 prompts", 8, 4, 2048, 120, 28, 4, ragged=True),
        # sixty-four users behind one system prompt
        attention("attention 1x64 system prompt", 1, 64, 8192, 256, 28, 4),
        # sixty-four answers to one long document: as many rows per key as make the products count
        attention("attention 1x64 document", 1, 64, 32768, 512, 40, 8),
        # beams of a float32 run
        attention("attention 5x8 float32", 5, 8, 1500, 60, 12, 2, dtype="float32", ragged=True),
        # many requests that share a little, some with nobody; small heads with sinks, larger pages
        attention("attention 48x5 small heads", 48, 5, 700, 90, 32, 8, head_dim=64, page=32, ragged=True, sinks=True),
        # the selection of one request, where few workgroups have anything to do
        select("select 1x4", 1, 4, 151936, 8),
        # sixteen requests, a grammar forbids a third of the tokens
        select("select 16x4 masked", 16, 4, 152064, 8, masked=3),
        # the most beams that a step of a busy engine brings
        select("select 64x8", 64, 8, 152064, 16),
        # many beams a request, a vocabulary that nothing divides
        select("select 7x24", 7, 24, 32003, 48),
        # keys' pages behind the shared ones: two requests of four beams, three pages a beam, in every layer
        reorder("reorder 2x4 pages", 2, 4, 3, 28, 4 * 16 * 128, "bfloat16"),
        # states of sixteen recurrent layers, eight requests of eight beams
        reorder("reorder 8x8 states", 8, 8, 1, 16, 32 * 64 * 64, "float32"),
    ]


def _spread(rng, low, high):
    """A whole number from ``low`` to ``high``, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _cost(case):
    """Bytes, or as many as are read while the products are worked."""
    need = work(case)
    return max(need["bytes"], need["flops"] / 50)


def draw(rng):
    op = rng.choice(["attention", "attention", "select", "reorder"])
    most = max(_cost(case) for case in listed())
    while True:
        if op == "attention":
            heads, kv_heads, head_dim = rng.choice([(12, 2, 128), (28, 4, 128), (40, 8, 128), (14, 2, 64), (32, 8, 64), (16, 4, 128), (8, 8, 96), (32, 2, 128)])
            case = attention(None, _spread(rng, 1, 48), _spread(rng, 1, 64), _spread(rng, 16, 32768), _spread(rng, 1, 1024), heads, kv_heads, head_dim,
                             rng.choice(["bfloat16", "bfloat16", "float32"]), rng.choice([8, 16, 32, 64]), rng.random() < 0.6, rng.random() < 0.3)
            if (case["groups"] * case["beams"] <= 256 and case["groups"] * case["beams"] * (case["shared"] + case["own"]) * kv_heads * head_dim <= 64 * 33280 * 8 * 128
                    and _cost(case) <= most):
                break
        elif op == "select":
            beams = _spread(rng, 1, 32)
            case = select(None, _spread(rng, 1, 64), beams, _spread(rng, 1000, 152064), rng.choice([beams, 2 * beams, 2 * beams, beams + 1]), rng.choice([0, 0, 2, 5]),
                          rng.random() < 0.2)
            if case["requests"] * beams <= 512 and (case["masked"] == 0 or case["vocab"] >= 8 * case["keep"]):
                break
        else:
            case = reorder(None, _spread(rng, 1, 32), _spread(rng, 2, 32), rng.choice([1, 1, 2, 5]), _spread(rng, 1, 28), _spread(rng, 64, 131072),
                           rng.choice(["bfloat16", "float32"]))
            if _cost(case) <= most:
                break
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ----------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Per group: how many sequences and shared keys; per sequence: how many keys in all."""
    sizes, shared, lens = [], [], []
    for g in range(case["groups"]):
        sizes.append(1 + (g * 5 + case["beams"] - 1) % case["beams"] if case["ragged"] else case["beams"])
        less = (g * 97) % (case["shared"] // 2 + 1) if case["ragged"] else 0
        shared.append(case["shared"] - less)
        for _ in range(sizes[-1]):
            lens.append(shared[-1] + 1 + (len(lens) * 61 + 17) % case["own"])
    return sizes, shared, lens


def _parents(case):
    """Every beam's parent: few beams have many children, as after a selection."""
    rng = random.Random(1000 * case["requests"] + case["beams"])
    return [[min(int(case["beams"] * rng.random() ** 2), case["beams"] - 1) for _ in range(case["beams"])] for _ in range(case["requests"])]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_attention(case, draw_normal, generator):
    dtype, page, heads, kv_heads, dim = DTYPES[case["dtype"]], case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    sizes, shared, lens = _lengths(case)
    width = -(-max(lens) // page)
    # pages in the order of a pool that has been in use for a while; a page that a prompt ends in is every beam's own
    needed = sum(s // page for s in shared) + sum(-(-n // page) - shared[g] // page for g, n in zip([g for g, k in enumerate(sizes) for _ in range(k)], lens))
    pages = needed + 9
    order = (torch.randperm(pages - 1, generator=generator) + 1).tolist()
    tables, copies, starts, at, b = [], [], [0], 0, 0
    for k, s in zip(sizes, shared):
        whole = s // page
        prefix, at = order[at:at + whole], at + whole
        first = len(tables)
        for _ in range(k):
            count = -(-lens[b] // page) - whole
            tables.append(prefix + order[at:at + count])
            if s % page and b > first:
                copies.append((tables[first][whole], order[at]))
            at, b = at + count, b + 1
        starts.append(b)
    k_cache = draw_normal((pages, kv_heads, page, dim)).to(dtype)
    v_cache = draw_normal((pages, kv_heads, dim, page)).to(dtype)
    if copies:
        source, target = (torch.tensor(x, device=DEVICE) for x in zip(*copies))
        k_cache[target], v_cache[target] = k_cache[source], v_cache[source]
    return dict(
        case=case, qkv=(2 * draw_normal((len(lens), (heads + 2 * kv_heads) * dim))).to(dtype), k_cache=k_cache, v_cache=v_cache,
        tables=_ints([t + [0] * (width - len(t)) for t in tables]), kv_lens=_ints(lens), group_starts=_ints(starts), shared_lens=_ints(shared),
        largest=max(sizes), longest=max(lens), scale=dim ** -0.5, sinks=draw_normal((heads,)) if case["sinks"] else None)


def _prepare_select(case, draw_normal, generator):
    requests, beams, vocab = case["requests"], case["beams"], case["vocab"]
    logits = 3 * draw_normal((requests * beams, vocab))
    if case["masked"]:
        forbidden = torch.rand((requests, 1, vocab), generator=generator).to(DEVICE) * case["masked"] < 1
        logits = logits.view(requests, beams, vocab).masked_fill_(forbidden, -math.inf).view(requests * beams, vocab)
    scores = -20 * torch.rand((requests, beams), generator=generator).to(DEVICE)
    if case["first"]:
        scores.fill_(-math.inf)[:, 0] = 0
    return dict(case=case, logits=logits, scores=scores)


def _prepare_reorder(case, draw_normal, generator):
    count = case["requests"] * case["beams"] * case["rows"]
    states = draw_normal((case["layers"], count + 5, case["width"])).to(DTYPES[case["dtype"]])
    slots = torch.randperm(count + 5, generator=generator)[:count].view(case["requests"], case["beams"], case["rows"])
    return dict(case=case, states=states, slots=slots.to(torch.int32).to(DEVICE), parents=_ints(_parents(case)))


def prepare(case, seed):
    generator = torch.Generator().manual_seed(seed)
    on_device = torch.Generator(DEVICE).manual_seed(seed)

    def draw_normal(shape):
        return torch.randn(shape, generator=on_device, device=DEVICE, dtype=torch.float32)

    return {"attention": _prepare_attention, "select": _prepare_select, "reorder": _prepare_reorder}[case["op"]](case, draw_normal, generator)


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _framework():
    """The kernels and the workspace that a program keeps."""
    from velox_amd.engine.batch import Workspace
    from velox_amd.kernels import load_ops

    return load_ops(DEVICE), Workspace(torch.device(DEVICE))


def _own(s):
    ops, workspace = _framework()
    case = s["case"]
    if case["op"] == "attention":
        return ops.shared_prefix_attention(s["qkv"], case["heads"], case["kv_heads"], case["head_dim"], s["k_cache"], s["v_cache"], case["page"], s["tables"], s["kv_lens"],
                                           s["group_starts"], s["shared_lens"], s["largest"], s["longest"], s["scale"], workspace, sinks=s["sinks"])
    if case["op"] == "select":
        return ops.beam_select(s["logits"], s["scores"], case["keep"])
    ops.reorder_states([s["states"]], s["slots"], s["parents"], axis=1)
    return s["states"]


def _plain_attention(s):
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    rows = s["qkv"].shape[0]
    n = torch.arange(s["longest"], device=DEVICE)
    page_of, offset = s["tables"].long()[:, n // page], n % page
    keys = s["k_cache"][page_of, :, offset].float().permute(0, 2, 3, 1).contiguous()  # [sequence, KV head, channel, key]
    scores = torch.matmul(s["qkv"][:, :heads * dim].float().view(rows, kv_heads, heads // kv_heads, dim), keys) * s["scale"]
    del keys
    scores = scores.masked_fill((n >= s["kv_lens"].view(-1, 1))[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].view(1, kv_heads, -1, 1) - top)
    values = s["v_cache"][page_of, :, :, offset].float().permute(0, 2, 1, 3).contiguous()  # [sequence, KV head, key, channel]
    return (torch.matmul(weights, values) / total).reshape(rows, heads * dim).to(s["qkv"].dtype)


def _plain_select(s):
    case, vocab = s["case"], s["logits"].shape[1]
    logits = s["logits"].double()  # (which candidate comes first hangs on differences far below a score's 32 bits)
    top = logits.amax(-1, keepdim=True)
    chances = logits - top - torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    values = s["scores"].double().view(-1, 1) + chances
    best, at = values.view(case["requests"], -1).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :case["keep"]], at[:, :case["keep"]]
    return best.float(), (at // vocab).to(torch.int32), (at % vocab).to(torch.int32)


def _plain_reorder(s):
    slots = s["slots"].long()
    sources = slots.gather(1, s["parents"].long()[:, :, None].expand_as(slots))
    s["states"][:, slots.view(-1)] = s["states"][:, sources.view(-1)]
    return s["states"]


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        sizes, shared, lens = _lengths(case)
        elem, per_key = DTYPES[case["dtype"]].itemsize, 2 * case["kv_heads"] * case["head_dim"]
        keys = sum(shared) + sum(lens) - sum(k * s for k, s in zip(sizes, shared))
        ends = 2 * len(lens) * case["heads"] * case["head_dim"]
        return {"bytes": elem * (keys * per_key + ends), "flops": 4 * case["head_dim"] * case["heads"] * sum(lens)}
    if case["op"] == "select":
        rows = case["requests"] * case["beams"]
        reading = case["requests"] if case["first"] else rows
        return {"bytes": 4 * reading * case["vocab"] + 4 * rows + 12 * case["requests"] * case["keep"], "flops": 3 * reading * case["vocab"]}
    moved = 0  # rows read or written
    for parents in _parents(case):
        changed = [p for j, p in enumerate(parents) if p != j]
        moved += len(changed) + len(set(changed))
    count = case["requests"] * case["beams"]
    return {"bytes": moved * case["rows"] * case["layers"] * case["width"] * DTYPES[case["dtype"]].itemsize + 4 * count * (case["rows"] + 1), "flops": 0}


def _exact_attention(s):
    """Sequence by sequence from the definition, its keys gathered one sequence at a time."""
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros((s["qkv"].shape[0], heads, dim), dtype=torch.float64, device=DEVICE)
    for b, length in enumerate(s["kv_lens"].tolist()):
        used = s["tables"][b, :-(-length // page)].long()
        keys = s["k_cache"][used].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :length].double()
        values = s["v_cache"][used].permute(1, 0, 3, 2).reshape(kv_heads, -1, dim)[:, :length].double()
        query = s["qkv"][b, :heads * dim].double().view(kv_heads, heads // kv_heads, dim)
        scores = s["scale"] * torch.matmul(query, keys.transpose(1, 2).contiguous())
        if s["sinks"] is not None:
            scores = torch.cat([scores, s["sinks"].double().view(kv_heads, -1, 1)], dim=2)
        out[b] = torch.matmul(torch.softmax(scores, dim=2)[:, :, :length].contiguous(), values).view(heads, dim)
    return out.view(-1, heads * dim)


def _exact_select(s):
    case, vocab = s["case"], s["logits"].shape[1]
    values = (torch.log_softmax(s["logits"].double(), dim=1) + s["scores"].double().view(-1, 1)).view(case["requests"], -1)
    best, at = torch.topk(values, case["keep"], dim=1)
    return best, torch.div(at, vocab, rounding_mode="floor").to(torch.int32), torch.remainder(at, vocab).to(torch.int32)


def exact(case, seed):
    if case["op"] == "reorder":
        return None  # (nothing is computed: the rows themselves move)
    state = prepare(case, seed)
    return _exact_attention(state) if case["op"] == "attention" else _exact_select(state)
