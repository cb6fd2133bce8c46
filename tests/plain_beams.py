"""Plain forms, in 64 bits and row by row, of the operators for several continuations of one prompt."""
import math

import torch


def shared_prefix_attention(qkv, num_heads, num_kv_heads, head_dim, k_cache, v_cache, block_size, block_tables, kv_lens, group_starts, shared_lens, scale, sinks=None):
    """Float64 ``[T, heads, dim]``: the outputs; the same with the values' magnitudes in the values' place; and float64 ``[T, heads]``: the
    largest sum of magnitudes behind a scaled score (what bounds the rounding of scores)."""
    group = num_heads // num_kv_heads
    num_seqs = kv_lens.shape[0]
    lens, starts, shared = kv_lens.tolist(), group_starts.tolist(), shared_lens.tolist()
    out = torch.zeros((num_seqs, num_heads, head_dim), dtype=torch.float64)
    size = torch.zeros_like(out)
    reach = torch.zeros((num_seqs, num_heads), dtype=torch.float64)
    k_cache, v_cache, tables, q = k_cache.cpu(), v_cache.cpu(), block_tables.cpu().long(), qkv.cpu()[:, :num_heads * head_dim].double().view(num_seqs, num_heads, head_dim)
    for b in range(num_seqs):
        if lens[b] <= 0:
            continue
        first, common = b, 0
        for g in range(len(shared)):
            if starts[g] <= b < starts[g + 1]:
                first, common = starts[g], min(shared[g], lens[starts[g]])
        if common > lens[b]:
            common = 0
        n = torch.arange(lens[b])
        page = torch.where(n < common, tables[first][(n // block_size).clamp(max=tables.shape[1] - 1)], tables[b][n // block_size])
        keys = k_cache[page, :, n % block_size].double()  # [keys, KV heads, dim]
        values = v_cache[page, :, :, n % block_size].double()
        for h in range(num_heads):
            kv = h // group
            scores = keys[:, kv] @ q[b, h] * scale
            reach[b, h] = (keys[:, kv].abs() @ q[b, h].abs()).max() * scale
            top = scores.max()
            weights = torch.exp(scores - top)
            denominator = weights.sum() + (0 if sinks is None else math.exp(float(sinks[h]) - float(top)))
            out[b, h] = weights @ values[:, kv] / denominator
            size[b, h] = weights @ values[:, kv].abs() / denominator
    return out, size, reach


def beam_values(logits, scores):
    """Float64 ``[requests, beams, vocab]``."""
    requests, beams = scores.shape
    x = logits.cpu().double().view(requests, beams, -1)
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    off = torch.where(x == top, 0.0, x - top)
    values = scores.cpu().double()[:, :, None] + (off - torch.exp(off).sum(-1, keepdim=True).log())
    nothing = (x == -math.inf) | ~(scores.cpu().double()[:, :, None] > -math.inf)
    return torch.where(nothing, -math.inf, values), torch.where(nothing, -math.inf, x)


def beam_select(logits, scores, keep):
    values, x = beam_values(logits, scores)
    requests, beams, vocab = values.shape
    out = []
    for r in range(requests):
        order = sorted(range(beams * vocab), key=lambda i: (-values[r].view(-1)[i].item(), i // vocab, -x[r].view(-1)[i].item(), i % vocab)) if beams * vocab < 3000 else None
        if order is None:  # (no two values of a long row are equal by accident: a stable sort by beam and logit, then by value)
            within = torch.sort(x[r], dim=-1, descending=True, stable=True).indices + torch.arange(beams)[:, None] * vocab
            within = within.view(-1)
            order = within[torch.sort(values[r].view(-1)[within], descending=True, stable=True).indices][:keep].tolist()
        out.append([(values[r].view(-1)[i].item(), i // vocab, i % vocab) for i in order[:keep]])
    best = torch.tensor([[c[0] for c in row] for row in out], dtype=torch.float64).view(requests, keep)
    parents = torch.tensor([[c[1] for c in row] for row in out], dtype=torch.int32).view(requests, keep)
    return best, parents, torch.tensor([[c[2] for c in row] for row in out], dtype=torch.int32).view(requests, keep)


def reorder_states(tensors, slots, parents, axis=0):
    """The tensors' new contents (the given ones are left alone)."""
    slots = slots.cpu()
    slots = slots[:, :, None] if slots.dim() == 2 else slots
    parents = parents.cpu().tolist()
    results = []
    for t in tensors:
        old, new = t.clone().movedim(axis, 0), t.clone()
        rows = new.movedim(axis, 0)
        for b in range(slots.shape[0]):
            for j, parent in enumerate(parents[b]):
                for p in range(slots.shape[2]):
                    to = int(slots[b, j, p])
                    source = int(slots[b, parent, p]) if 0 <= parent < slots.shape[1] else -1
                    if 0 <= to < rows.shape[0] and 0 <= source < rows.shape[0]:
                        rows[to] = old[source]
        results.append(new)
    return results
