"""Attention over shared prefixes, selection over beams and the states' change of places against their plain forms in 64 bits."""
import math

import pytest
import torch

import plain_beams as plain
from velox_amd.engine.batch import Workspace

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from velox_amd.kernels import load_ops

    return load_ops("cuda")


@pytest.fixture()
def workspace():
    return Workspace(torch.device("cuda"))


# ----------------------------------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------------------------------
class Batch:
    """Sequences in groups over a cache.  ``groups``: (sequences, shared keys) each; ``lens``: keys of every sequence, or how many each has of
    its own.  All that nobody may read is no number: pages in nobody's hands, places behind a sequence's end, the shared keys' places in
    the pages of all but a group's first sequence; table entries that nobody may look at lead to such a page."""

    def __init__(self, dtype, heads, kv_heads, dim, page, groups, lens, before=0, behind=0, seed=0, with_kv=True, sinks=False, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.args = (heads, kv_heads, dim)
        self.page = page
        starts, shared, first_of = [before], [], {}
        for count, keys in groups:
            for b in range(starts[-1], starts[-1] + count):
                first_of[b] = (starts[-1], keys)
            starts.append(starts[-1] + count)
            shared.append(keys)
        num = starts[-1] + behind
        assert len(lens) == num
        width = max(-(-max(lens) // page), 1050 // page) + 1
        wild = 0
        tables = torch.full((num, width), wild, dtype=torch.int32)
        pages = 1 + sum(-(-n // page) for n in lens) + 3
        order = (torch.randperm(pages - 1, generator=g) + 1).tolist()
        k = torch.full((pages, kv_heads, page, dim), math.nan)
        v = torch.full((pages, kv_heads, dim, page), math.inf)
        at = 0
        for b, n in enumerate(lens):
            first, common = first_of.get(b, (b, 0))
            common = 0 if first == b else min(common, lens[first])
            if common > n:
                common = 0
            for p in range(-(-n // page)):
                lo, hi = max(p * page, common), min((p + 1) * page, n)
                if hi <= lo:
                    continue  # (shared keys alone: not looked at)
                tables[b, p] = order[at]
                at += 1
                k[tables[b, p], :, lo - p * page:hi - p * page] = torch.randn((kv_heads, hi - lo, dim), generator=g) * spread
                v[tables[b, p], :, :, lo - p * page:hi - p * page] = torch.randn((kv_heads, dim, hi - lo), generator=g)
        channels = (heads + 2 * kv_heads if with_kv else heads) * dim
        self.qkv = torch.randn((num, channels), generator=g).to(dtype).cuda()
        self.k, self.v = k.to(dtype).cuda(), v.to(dtype).cuda()
        self.tables, self.lens = tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
        self.starts, self.shared = torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(shared, dtype=torch.int32).cuda()
        self.largest = max([c for c, _ in groups], default=1)
        self.most_keys = max(lens)
        self.longest = max(max(lens), 1050)  # (keys enough to be shared out among workgroups)
        self.scale = dim ** -0.5
        self.sinks = torch.randn(heads, generator=g).cuda() if sinks else None

    def run(self, ops, workspace, **changed):
        largest, longest = changed.get("largest", self.largest), changed.get("longest", self.longest)
        return ops.shared_prefix_attention(self.qkv, *self.args, self.k, self.v, self.page, self.tables, self.lens, self.starts, self.shared, largest, longest, self.scale,
                                           workspace, sinks=self.sinks)

    def check(self, got):
        heads, kv_heads, dim = self.args
        want, size, reach = plain.shared_prefix_attention(self.qkv, *self.args, self.k, self.v, self.page, self.tables, self.lens, self.starts, self.shared, self.scale, self.sinks)
        # A score is a sum of `dim` products in float32, off by at most dim 2^-24 of the sum of their magnitudes, and the scaling and the exponent's
        # argument by 2^-24 of it each; a relative error of the weights twice that (numerator and denominator).  Exponentials and sums of up to
        # n weights or weighted values, joined once: (n + 64) 2^-24, and 2^-21 for each of exp (two, the joining's among them).  In bfloat16 a weight is
        # rounded before its product (2^-8 of the values' magnitudes) and so is the result (2^-8 of it); float32 results by 2^-24.
        n = max(self.most_keys, 1)
        weights = 2 * (dim + 4) * 2.0 ** -24 * reach[:, :, None] + (n + 64) * 2.0 ** -24 + 2 * 2.0 ** -21
        rounding = 2.0 ** -8 if self.qkv.dtype == BF16 else 2.0 ** -24
        allowed = size * (weights + (2.0 ** -8 if self.qkv.dtype == BF16 else 0)) * 1.01 + rounding * want.abs() * 1.01 + 1e-30
        off = (got.cpu().double().view_as(want) - want).abs()
        assert torch.isfinite(got).all(), "something that nobody may read was read"
        worst = (off / allowed).max().item()
        assert worst <= 1, f"{worst} of what is allowed"
        return worst


def own(count, shared, low, high, step=7):
    return [shared + low + (i * step) % (high - low + 1) for i in range(count)]


SHAPES = [
    # heads, KV heads, head size, page
    (12, 2, 128, 16), (4, 4, 64, 8), (7, 1, 16, 16), (6, 2, 48, 32), (5, 1, 80, 64), (8, 2, 96, 16), (4, 2, 192, 8), (3, 1, 256, 16), (34, 2, 32, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_shapes(ops, workspace, dtype, shape):
    """Two groups (a shared length that ends inside a page, one that ends with it), sequences before, between and behind them."""
    lens = [37, 1] + own(5, 203, 1, 90) + own(3, 64, 0, 40) + [130]
    b = Batch(dtype, *shape, groups=[(5, 203), (3, 64)], lens=lens, before=2, behind=1)
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("shared", [1, 7, 8, 31, 32, 33, 127, 128, 129, 500])
def test_attention_shared_lengths(ops, workspace, dtype, page, shared):
    b = Batch(dtype, 4, 2, 64, page, groups=[(3, shared)], lens=[shared + 1, shared + 40, shared + 2], seed=shared)
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_edges_of_groups(ops, workspace, dtype):
    """No keys; as many as are shared; fewer than are shared; a group whose first sequence has fewer keys than it is said to share; groups of one and of none."""
    groups = [(4, 50), (3, 90), (1, 64), (0, 33), (2, 0), (2, 20)]
    lens = [50, 51, 49, 0] + [70, 75, 71] + [80] + [5, 6] + [0, 30]
    b = Batch(dtype, 4, 2, 64, 16, groups=groups, lens=lens)
    got = b.run(ops, workspace)
    b.check(got)
    assert (got[3] == 0).all() and (got[10] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("count", [1, 2, 9, 10, 19, 37, 64])
def test_attention_group_sizes(ops, workspace, dtype, count):
    """One to several blocks of rows, with queries alone in their rows and a sink."""
    b = Batch(dtype, 14, 2, 64, 16, groups=[(count, 300)], lens=own(count, 300, 1, 33), with_kv=False, sinks=True, seed=count)
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_long(ops, workspace, dtype):
    """Keys over many workgroups, of the shared part and of one sequence's own."""
    b = Batch(dtype, 8, 4, 128, 16, groups=[(3, 5003), (2, 41)], lens=[5010, 9001, 5004] + [42, 2500] + [3], behind=1)
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,count,shared", [(28, 4, 128, 20, 2048), (10, 2, 128, 64, 1500), (28, 4, 64, 40, 3001), (8, 1, 128, 17, 8192)])
def test_attention_many_rows(ops, workspace, dtype, heads, kv_heads, dim, count, shared):
    """Several blocks of many rows over many tiles, the last block in part; the same bits every time."""
    b = Batch(dtype, heads, kv_heads, dim, 16, groups=[(count, shared), (2, 100)], lens=own(count, shared, 1, 150) + [120, 101], seed=count)
    first = b.run(ops, workspace)
    b.check(first)
    for _ in range(50):
        assert torch.equal(first, b.run(ops, workspace))


def test_attention_more_sequences_than_are_held(ops, workspace):
    """More than 1,024 sequences, in groups and not."""
    groups = [(1 + g % 4, 5 + g % 60) for g in range(520)]
    lens = [s + 1 + (i % 3) for i, s in enumerate(s for c, s in groups for _ in range(c))]
    b = Batch(BF16, 2, 1, 16, 8, groups=groups, lens=lens + [7] * 20, behind=20)
    first = b.run(ops, workspace)
    b.check(first)
    for _ in range(10):
        assert torch.equal(first, b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_many_sequences_and_groups(ops, workspace, dtype):
    """More than 64 of both (a wave's lanes), most of them short."""
    groups = [(1 + g % 3, 9 + g) for g in range(70)]
    lens = [s + 1 + (i % 5) for i, s in enumerate(s for c, s in groups for _ in range(c))]
    b = Batch(dtype, 2, 1, 32, 8, groups=groups, lens=[4] * 3 + lens, before=3)
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [128, 1024, 65536])
@pytest.mark.parametrize("count,shared", [(3, 300), (70, 4100)])
def test_attention_large_pages(ops, workspace, dtype, page, count, shared):
    b = Batch(dtype, 8, 2, 64, page, groups=[(count, shared)], lens=own(count, shared, 1, 40))
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("longest", [0, 1, 31, 64, 127, 130])
def test_attention_lengths_beyond_the_most(ops, workspace, dtype, longest):
    """They count as the most that was said, a group's shared keys among them."""
    b = Batch(dtype, 8, 2, 64, 16, groups=[(5, 128)], lens=own(5, 128, 1, 40) + [200, 3], behind=2)
    got = b.run(ops, workspace, longest=longest)
    b.lens = b.lens.clamp(max=longest)
    b.check(got)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("count,shared", [(3, 300), (12, 1000), (63, 4200)])
def test_attention_planned_ahead(ops, workspace, dtype, count, shared):
    """More than 64 sequences or groups are planned by a kernel of its own, to the same items: others without a key, or groups without a
    sequence, change nothing for the rows that were there."""
    few = Batch(dtype, 28, 4, 128, 16, groups=[(count, shared)], lens=own(count, shared, 1, 300))
    want = few.run(ops, workspace)
    few.check(want)
    many = Batch(dtype, 28, 4, 128, 16, groups=[(count, shared)], lens=own(count, shared, 1, 300) + [0] * (65 - count), behind=65 - count)
    many.qkv[:count], many.k, many.v, many.tables[:count] = few.qkv, few.k, few.v, few.tables
    for _ in range(20):
        got = many.run(ops, workspace)
        assert torch.equal(got[:count], want) and not got[count:].any()
    few.starts, few.shared = torch.cat([few.starts, few.starts[-1:].repeat(64)]), torch.cat([few.shared, few.shared.repeat(64)])
    for _ in range(20):
        assert torch.equal(few.run(ops, workspace), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups", [61, 63, 64, 65, 127, 128, 129])
def test_attention_about_a_waves_lanes(ops, workspace, dtype, groups):
    sizes = [(1 + g % 3, 10 + 37 * (g % 7)) for g in range(groups)]
    lens = [length for g, (count, shared) in enumerate(sizes) for length in own(count, shared, g % 2, 30)]
    b = Batch(dtype, 4, 2, 64, 16, groups=sizes, lens=lens)
    b.check(b.run(ops, workspace))
    b = Batch(dtype, 4, 2, 64, 16, groups=[(2, 40)], lens=own(2, 40, 1, 9) + [7 * (i % 9) for i in range(groups - 2)], behind=groups - 2)
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("beyond", [0, 1, 7, 8, 9, 33, 63])
def test_attention_many_rows_of_any_end(ops, workspace, dim, beyond):
    """Shared keys that end anywhere in a tile; the first sequence has none of its own, and what lies behind its last key is no number."""
    shared = 4096 + beyond
    b = Batch(BF16, 8, 2, dim, 16, groups=[(70, shared)], lens=own(70, shared, 0, 40))
    assert ops._shared_prefix_shape(ops.num_cus, 70, 1, 8, 2, dim, 2, 70, b.longest)[0] == 8
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("heads,kv_heads,dim,groups,own_most", [
    (16, 4, 64, [(37, 2500)], 150), (16, 4, 128, [(36, 2300), (3, 70), (1, 5)], 700), (8, 8, 32, [(40, 4200), (2, 33)], 60), (32, 8, 96, [(20, 2600)], 90),
    (12, 2, 128, [(70, 2000)], 120), (12, 2, 128, [(50, 2001), (31, 1000)], 60), (8, 4, 16, [(4, 700), (61, 3100)] + [(2, 90)] * 9, 200), (14, 2, 80, [(13, 4300)] * 6, 40),
])
@pytest.mark.parametrize("sinks", [False, True])
def test_attention_single_float32_row_tiles_of_many_steps(ops, workspace, heads, kv_heads, dim, groups, own_most, sinks):
    """Two workgroups to a compute unit, with up to 64 sequences and with more; odd and even numbers of row tiles; the same bits every time."""
    lens = [n for count, shared in groups for n in own(count, shared, 0, own_most)]
    b = Batch(F32, heads, kv_heads, dim, 16, groups=groups, lens=lens, sinks=sinks, seed=heads)
    assert ops._shared_prefix_shape(ops.num_cus, len(lens), len(groups), heads, kv_heads, dim, 4, b.largest, b.longest)[:2] == (1, 2 * ops.num_cus // kv_heads)
    first = b.run(ops, workspace)
    b.check(first)
    for _ in range(10):
        assert torch.equal(first, b.run(ops, workspace))


def test_attention_scratch_is_what_it_says_of_many_sequences(ops):
    """Items written down ahead, in a workspace of the stated size that is fixed."""
    for heads, kv_heads, dim, groups, own_most in ((12, 2, 128, [(70, 2000)], 120), (8, 4, 16, [(4, 700), (61, 3100)] + [(2, 90)] * 9, 200)):
        lens = [n for count, shared in groups for n in own(count, shared, 0, own_most)]
        workspace = Workspace(torch.device("cuda"))
        workspace.reserve("shared_prefix_parts", ops.shared_prefix_scratch_elems(heads, kv_heads, dim, len(lens), len(groups)))
        workspace.fix()
        for dtype in (F32, BF16):
            b = Batch(dtype, heads, kv_heads, dim, 16, groups=groups, lens=lens)
            b.check(b.run(ops, workspace))


def test_attention_without_groups(ops, workspace):
    b = Batch(BF16, 12, 2, 128, 16, groups=[], lens=[100, 1, 333], behind=3)
    b.check(b.run(ops, workspace))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_peaked_scores(ops, workspace, dtype):
    """Scores far apart: the running maximum moves late, most weights vanish."""
    b = Batch(dtype, 12, 2, 128, 16, groups=[(6, 700)], lens=own(6, 700, 1, 200), spread=6.0)
    b.check(b.run(ops, workspace))


def test_attention_result_does_not_hang_on_the_bounds(ops, workspace):
    """The largest group and the most keys may be said too large; a call repeated gives the same bits."""
    b = Batch(F32, 12, 2, 128, 16, groups=[(3, 450), (1, 3)], lens=own(3, 450, 1, 50) + [90])
    first = b.run(ops, workspace)
    assert torch.equal(first, b.run(ops, workspace))
    b.check(b.run(ops, workspace, largest=4, longest=b.tables.shape[1] * 16))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("shared", [1, 31, 32, 33, 64, 129, 200])
def test_attention_few_keys(ops, workspace, dtype, shape, shared):
    """A workgroup takes all of a sequence's keys."""
    lens = [37, 1, 0] + own(5, shared, 0, 50) + own(3, 64, 1, 40) + [min(shared, 20), 130]
    b = Batch(dtype, *shape, groups=[(5, shared), (4, 64)], lens=lens, before=3, behind=1, sinks=shared % 2 == 1)
    assert ops._shared_prefix_shape(ops.num_cus, 13, 2, *shape[:3], 4 if dtype == F32 else 2, 5, b.most_keys)[0] == 0
    for largest in (5, 13):
        b.check(b.run(ops, workspace, largest=largest, longest=b.most_keys))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_few_keys_of_many_groups(ops, workspace, dtype):
    sizes = [(1 + g % 3, 3 + 5 * (g % 7)) for g in range(200)]
    lens = [length for g, (count, shared) in enumerate(sizes) for length in own(count, shared, g % 2, 30)]
    b = Batch(dtype, 4, 2, 64, 16, groups=sizes, lens=lens)
    assert ops._shared_prefix_shape(ops.num_cus, len(lens), 200, 4, 2, 64, 4 if dtype == F32 else 2, 3, b.most_keys)[0] == 0
    b.check(b.run(ops, workspace, longest=b.most_keys))
    b.check(b.run(ops, workspace))


def test_attention_few_keys_of_a_group_larger_than_said(ops, workspace):
    """What a group has beyond the largest reads its own pages alone."""
    b = Batch(BF16, 12, 2, 128, 16, groups=[(6, 100)], lens=own(6, 100, 1, 60))
    b.tables[4:, :100 // 16] = b.tables[0, :100 // 16]  # (their own tables lead to the shared keys as well)
    last = b.tables[4:, 100 // 16].tolist()
    for page in last:
        b.k[page, :, :100 % 16] = b.k[b.tables[0, 100 // 16], :, :100 % 16]
        b.v[page, :, :, :100 % 16] = b.v[b.tables[0, 100 // 16], :, :, :100 % 16]
    want = b.run(ops, workspace, longest=b.most_keys)
    b.check(want)
    assert torch.equal(b.run(ops, workspace, largest=4, longest=b.most_keys)[:4], want[:4])
    b.check(b.run(ops, workspace, largest=4, longest=b.most_keys))


def test_attention_group_larger_than_said(ops, workspace):
    """What a group has beyond ``largest_group`` reads all its keys through its own table."""
    b = Batch(BF16, 12, 2, 128, 16, groups=[(4, 0), (5, 0)], lens=own(4, 450, 1, 50) + own(5, 90, 1, 50))
    b.shared.copy_(torch.tensor([440, 80], dtype=torch.int32))
    b.tables[1, :27] = b.tables[0, :27]  # (the first two of either share whole pages in earnest; the others have pages of their own)
    b.tables[5, :5] = b.tables[4, :5]
    b.k[b.tables[1, 27].long(), :, :8], b.v[b.tables[1, 27].long(), :, :, :8] = b.k[b.tables[0, 27].long(), :, :8], b.v[b.tables[0, 27].long(), :, :, :8]
    got = b.run(ops, workspace, largest=2)
    b.starts, b.shared = torch.tensor([0, 2, 4, 6], dtype=torch.int32).cuda(), torch.tensor([440, 0, 80], dtype=torch.int32).cuda()
    b.check(got)


def test_attention_agrees_with_paged_attention(ops, workspace):
    """Tables that are filled in full: the same answers as the kernels that read every sequence's keys."""
    g = torch.Generator().manual_seed(5)
    heads, kv_heads, dim, page, count, shared = 28, 4, 128, 16, 6, 20 * 16
    lens = own(count, shared, 1, 100)
    width = -(-max(lens) // page)
    tables = torch.randperm(1000, generator=g)[:count * width].view(count, width).to(torch.int32)
    tables[:, :shared // page] = tables[0, :shared // page]
    k = torch.randn((1000, kv_heads, page, dim), generator=g).to(BF16).cuda()
    v = torch.randn((1000, kv_heads, dim, page), generator=g).to(BF16).cuda()
    qkv = torch.randn((count, (heads + 2 * kv_heads) * dim), generator=g).to(BF16).cuda()
    tables, lens_dev = tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    cu = torch.arange(count + 1, dtype=torch.int32).cuda()
    want = ops.paged_attention(qkv, heads, kv_heads, dim, k, v, page, tables, cu, lens_dev, 1, max(lens), dim ** -0.5, None, True, workspace)
    starts, common = torch.tensor([0, count], dtype=torch.int32).cuda(), torch.tensor([shared], dtype=torch.int32).cuda()
    got = ops.shared_prefix_attention(qkv, heads, kv_heads, dim, k, v, page, tables, lens_dev, starts, common, count, max(lens), dim ** -0.5, workspace)
    # two results that each are off by 2^-8 of the weighted magnitudes (about 1 here at most) and by a rounding of 2^-8 of themselves
    torch.testing.assert_close(got.float(), want.float(), rtol=2 * 2.0 ** -8, atol=2 * 2.0 ** -8)


@pytest.mark.parametrize("most", [256, 1050])
def test_attention_captured(ops, most):
    """A captured call replays with other lengths, other groups and other pages' contents, with eager calls of the same workspace between."""
    workspace = Workspace(torch.device("cuda"))
    a = Batch(F32, 8, 2, 64, 16, groups=[(3, 200), (2, 70)], lens=own(3, 200, 1, 60) + own(2, 70, 1, 50), seed=1)
    other = Batch(F32, 8, 2, 64, 16, groups=[(2, 100), (3, 33)], lens=own(2, 100, 1, 150) + own(3, 33, 1, 220), seed=2)
    width = max(a.tables.shape[1], other.tables.shape[1])
    pages = max(a.k.shape[0], other.k.shape[0])
    for b in (a, other):
        b.tables = torch.nn.functional.pad(b.tables, (0, width - b.tables.shape[1]))
        b.k = torch.cat([b.k, torch.full_like(b.k[:1], math.nan).expand(pages - b.k.shape[0], -1, -1, -1)]) if b.k.shape[0] < pages else b.k
        b.v = torch.cat([b.v, torch.full_like(b.v[:1], math.nan).expand(pages - b.v.shape[0], -1, -1, -1)]) if b.v.shape[0] < pages else b.v
        b.largest, b.longest = 3, most
    names = ("qkv", "k", "v", "tables", "lens", "starts", "shared")
    live = {name: getattr(a, name).clone() for name in names}

    def call():
        return ops.shared_prefix_attention(live["qkv"], *a.args, live["k"], live["v"], 16, live["tables"], live["lens"], live["starts"], live["shared"], 3, most, a.scale, workspace)

    call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = call()
    for round in range(3):
        for b in (other, a):
            for name in names:
                live[name].copy_(getattr(b, name))
            eager = call()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(result, eager)
            b.check(result.clone())


def test_attention_captured_of_many_sequences(ops):
    """Two captured calls that share a workspace, planned ahead, replayed in turn with other lengths and groups, eager calls between."""
    workspace = Workspace(torch.device("cuda"))
    made = []
    for count, dtype in ((70, BF16), (90, F32)):
        most = 400
        groups = [(5, 100 + 3 * g) for g in range(count // 5)]
        first = Batch(dtype, 8, 2, 64, 16, groups=groups, lens=[n for g in range(count // 5) for n in own(5, 100 + 3 * g, 1, 60)])
        second = Batch(dtype, 8, 2, 64, 16, groups=groups[:-1] + [(5, 0)], lens=[n for g in range(count // 5) for n in own(5, 100 + 3 * g, 0, 40)], seed=3)
        live = {name: getattr(first, name).clone() for name in ("qkv", "tables", "lens", "starts", "shared")}
        pages = max(first.k.shape[0], second.k.shape[0])
        for b in (first, second):
            spare = pages - b.k.shape[0]
            b.k, b.v = (torch.cat([t, torch.full_like(t[:1], math.nan).expand(spare, -1, -1, -1)]) if spare else t for t in (b.k, b.v))
        live["k"], live["v"] = first.k.clone(), first.v.clone()

        def call(live=live, args=first.args, scale=first.scale, largest=first.largest):
            return ops.shared_prefix_attention(live["qkv"], *args, live["k"], live["v"], 16, live["tables"], live["lens"], live["starts"], live["shared"], largest, 1050, scale, workspace)

        made.append([first, second, live, call])
    for _, _, _, call in made:
        call()
    torch.cuda.synchronize()
    for m in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            m.append(m[3]())
        m.append(graph)
    for round in range(4):
        for first, second, live, call, result, graph in made:
            b = (first, second)[round % 2]
            for name, t in live.items():
                t.copy_(getattr(b, name))
            graph.replay()
            eager = call()
            torch.cuda.synchronize()
            assert torch.equal(result, eager)
            b.check(eager)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("count,shared,own_most", [(3, 100, 30), (4, 900, 200), (70, 4100, 40)])
def test_attention_pages_beyond_32_bits(ops, workspace, dtype, count, shared, own_most):
    """The same bits from pages whose offsets in bytes and in elements pass 32 bits."""
    b = Batch(dtype, 8, 2, 128, 16, groups=[(count, shared)], lens=own(count, shared, 1, own_most))
    longest = b.most_keys if shared < 200 else b.longest  # (few keys are taken whole)
    want = b.run(ops, workspace, longest=longest)
    b.check(want)
    pages = b.k.shape[0]
    many = 2 ** 32 // (2 * 16 * 128) + pages + 1  # (2^32 elements and more)
    k, v = torch.empty((many,) + b.k.shape[1:], dtype=dtype, device="cuda"), torch.empty((many,) + b.v.shape[1:], dtype=dtype, device="cuda")
    k[many - pages:], v[many - pages:] = b.k, b.v
    b.k, b.v, b.tables = k, v, b.tables + (many - pages)
    assert torch.equal(b.run(ops, workspace, longest=longest), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("count,shared,own_most", [(3, 100, 30), (4, 900, 200), (40, 3000, 60), (70, 4100, 40)])
def test_attention_infinite_values(ops, workspace, dtype, count, shared, own_most):
    """An infinite value makes its channel infinite for those who see it, not a number that is none, and nothing else."""
    b = Batch(dtype, 8, 2, 64, 16, groups=[(count, shared)], lens=own(count, shared, 2, own_most), spread=0.2)
    b.longest = max(b.most_keys, 1050) if shared > 200 else b.most_keys
    want = b.run(ops, workspace).view(count, 2, 4, 64)
    for key in (0, shared - 1):
        b.v[b.tables[0, key // 16].long(), 1, 7, key % 16] = math.inf  # (a shared key of the second KV head)
    last = b.lens[2].item() - 1
    b.v[b.tables[2, last // 16].long(), 0, 5, last % 16] = -math.inf  # (one of the third sequence's own, of the first)
    got = b.run(ops, workspace).view(count, 2, 4, 64)
    assert (got[:, 1, :, 7] == math.inf).all() and (got[2, 0, :, 5] == -math.inf).all()
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[:, 1, :, 7] = rest[2, 0, :, 5] = False
    assert torch.equal(got[rest], want[rest])


def test_attention_on_another_stream(ops, workspace):
    b = Batch(BF16, 12, 2, 128, 16, groups=[(6, 700)], lens=own(6, 700, 1, 200))
    want = b.run(ops, workspace)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = b.run(ops, Workspace(torch.device("cuda")))
    stream.synchronize()
    assert torch.equal(want, got)


def test_attention_scratch_is_what_it_says(ops):
    """A workspace of the stated size, fixed, serves every step within its limits."""
    for heads, kv_heads, dim, page in SHAPES:
        workspace = Workspace(torch.device("cuda"))
        workspace.reserve("shared_prefix_parts", ops.shared_prefix_scratch_elems(heads, kv_heads, dim, 40, 6))
        workspace.fix()
        for dtype in (BF16, F32):
            for groups, lens, behind in ([(40, 33)], own(40, 33, 1, 3), 0), ([(2, 100)] * 6, own(12, 100, 1, 3), 0), ([], [5], 1):
                b = Batch(dtype, heads, kv_heads, dim, page, groups=groups, lens=lens, behind=behind)
                b.run(ops, workspace)
    torch.cuda.synchronize()


# ----------------------------------------------------------------------------------------------------------------------
# selection
# ----------------------------------------------------------------------------------------------------------------------
def check_selection(ops, logits, scores, keep):
    values, parents, tokens = ops.beam_select(logits.cuda(), scores.cuda(), keep)
    want, want_parents, want_tokens = plain.beam_select(logits, scores, keep)
    assert torch.equal(parents.cpu(), want_parents) and torch.equal(tokens.cpu(), want_tokens)
    # values are worked in 64 bits (to 1e-10 or so of the sums) and rounded once
    got = values.cpu().double()
    assert torch.equal(got == -math.inf, want == -math.inf)
    finite = want > -math.inf
    assert ((got - want).abs()[finite] <= 2.0 ** -24 * want.abs()[finite] + 1e-9).all()


def random_case(requests, beams, vocab, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((requests * beams, vocab), generator=g) * spread, -10 * torch.rand((requests, beams), generator=g)


@pytest.mark.parametrize("requests,beams,vocab,keep", [
    (1, 4, 151936, 8), (3, 2, 32003, 4), (2, 7, 2047, 14), (2, 7, 2049, 14), (1, 1, 8192, 1), (1, 1, 8193, 64), (5, 3, 17, 6), (2, 4, 1, 4), (1, 1, 1, 1), (1, 64, 3, 64),
    (2, 33, 4099, 33), (1, 200, 1021, 64), (1, 256, 9000, 2), (40, 2, 9001, 4), (3, 24, 32003, 48),
])
def test_select_sizes(ops, requests, beams, vocab, keep):
    check_selection(ops, *random_case(requests, beams, vocab, seed=vocab), keep)


def test_select_busy_step(ops):
    """Rows enough for the large pieces."""
    check_selection(ops, *random_case(16, 8, 40000), 16)


@pytest.mark.parametrize("vocab", [50, 5000, 20011])
def test_select_masked(ops, vocab):
    """Rows with nothing allowed, with one token, with fewer than are wanted; no numbers; the type's lowest value."""
    logits, scores = random_case(5, 4, vocab)
    allowed = torch.rand((20, vocab), generator=torch.Generator().manual_seed(1)) < 0.5
    allowed[0:4] = False
    allowed[4:8] = False
    allowed[4, vocab - 1] = allowed[6, 3] = True
    allowed[8] = False
    logits = logits.masked_fill(~allowed, -math.inf)
    logits[12, 5] = math.nan
    logits[13] = math.nan
    logits[16:20] = torch.where(allowed[16:20], logits[16:20], torch.finfo(F32).min)
    check_selection(ops, logits, scores, 8)


@pytest.mark.parametrize("vocab", [50, 9000])
def test_select_beams_that_are_not_there(ops, vocab):
    logits, scores = random_case(4, 6, vocab)
    scores[0, 1:] = -math.inf
    scores[1] = -math.inf
    scores[2, 0] = scores[2, 5] = -math.inf
    scores[3, 2] = math.nan
    logits[6 + 2] = math.nan
    check_selection(ops, logits, scores, 12)


@pytest.mark.parametrize("absent", [range(0, 100), range(100, 200), range(0, 200, 2)])
def test_select_many_lists_of_which_many_are_empty(ops, absent):
    logits, scores = random_case(2, 200, 1021)
    scores[1, list(absent)] = -math.inf
    check_selection(ops, logits, scores, 64)


@pytest.mark.parametrize("keep", [4, 16, 17, 64])
def test_select_most_of_a_piece_alike(ops, keep):
    """More equal ones than are ranked: places decide."""
    g = torch.Generator().manual_seed(4)
    logits = torch.zeros((6, 20000))
    logits[1] = (torch.arange(20000) > 12000).float()
    logits[2, 5000:] = -math.inf
    logits[3, ::2] = 1.0
    logits[4] = torch.randn(20000, generator=g).round()
    check_selection(ops, logits, torch.zeros((3, 2)), keep)


@pytest.mark.parametrize("vocab,keep", [(40, 10), (2500, 64), (9001, 20)])
def test_select_ties(ops, vocab, keep):
    """Equal logits in a row, equal rows, zeros of both signs."""
    g = torch.Generator().manual_seed(2)
    logits = torch.randint(-2, 3, (12, vocab), generator=g).float()
    logits[3] = logits[4]
    logits[0] = 0.0
    logits[1] = torch.where(torch.arange(vocab) % 3 == 0, -0.0, 0.0)
    logits[6:9] = logits[6]
    scores = torch.zeros((4, 3))
    scores[3] = torch.tensor([-1.0, -1.0, -2.0])
    check_selection(ops, logits, scores, keep)


def test_select_infinite_and_far_logits(ops):
    logits, scores = random_case(3, 2, 3000)
    logits[0, 77] = math.inf
    logits[1, 5] = logits[1, 2999] = math.inf
    logits[2] *= 1000
    logits[4] -= 1e6
    check_selection(ops, logits, scores, 5)


@pytest.mark.parametrize("vocab", [3000, 40000])
@pytest.mark.parametrize("about,spread", [(1e4, 400.0), (5e8, 100.0), (2.0 ** 30, 500.0), (2e9, 300.0), (1.7e10, 3000.0), (-1.7e10, 3000.0), (0.0, 1e30), (3e38, 3e36)])
def test_select_logits_of_any_size(ops, vocab, about, spread):
    """Where neighbouring numbers of 32 bits are further apart than exponentials reach, too."""
    logits, scores = random_case(2, 3, vocab, seed=9, spread=spread)
    check_selection(ops, logits + about, scores, 7)


def test_select_rising_logits(ops):
    """What a row's sum refers to moves again and again."""
    logits = torch.linspace(-1.0, 1.0, 30000)[None] * torch.tensor([10.0, 2e3, 1e5, 1e9, 1e12, 3e38])[:, None]
    check_selection(ops, logits, torch.zeros((3, 2)), 9)
    check_selection(ops, logits.flip(1).contiguous(), torch.zeros((2, 3)), 9)


def test_select_infinite_scores(ops):
    """Every continuation is named once, also where infinity less infinity would be its worth."""
    logits, scores = random_case(2, 3, 3000)
    scores[:, 1] = math.inf
    logits[1, 9] = math.inf
    values, parents, tokens = (t.cpu() for t in ops.beam_select(logits.cuda(), scores.cuda(), 12))
    assert values[0, 0] == math.inf and (parents[0, 0], tokens[0, 0]) == (1, 9) and (values[1] == math.inf).all() and (parents[1] == 1).all()
    for r in range(2):
        assert len(set(zip(parents[r].tolist(), tokens[r].tolist()))) == 12
    best = torch.sort(logits[4], descending=True, stable=True).indices[:12]
    assert tokens[1].tolist() == best.tolist()
    rest = torch.sort((torch.log_softmax(logits.double(), 1)[:3] + scores[0].double()[:, None])[[0, 2]].view(-1), descending=True).values[:11]
    assert ((values[0, 1:].double() - rest).abs() <= 2.0 ** -24 * rest.abs() + 1e-9).all()


def test_select_rows_anywhere(ops):
    """Rows that begin at any multiple of four bytes."""
    logits, scores = random_case(2, 3, 10007)
    for shift in (1, 2, 3):
        room = torch.zeros(logits.numel() + 4, device="cuda")
        room[shift:shift + logits.numel()] = logits.view(-1).cuda()
        moved = room[shift:shift + logits.numel()].view_as(logits)
        values, parents, tokens = ops.beam_select(moved, scores.cuda(), 6)
        again = ops.beam_select(logits.cuda(), scores.cuda(), 6)
        assert torch.equal(values, again[0]) and torch.equal(parents, again[1]) and torch.equal(tokens, again[2])
    check_selection(ops, logits, scores, 6)


def test_select_captured(ops):
    logits, scores = random_case(3, 4, 20000)
    live, at = logits.cuda(), scores.cuda()
    ops.beam_select(live, at, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = ops.beam_select(live, at, 8)
    for seed in range(3):
        x, y = random_case(3, 4, 20000, seed=seed + 5)
        live.copy_(x)
        at.copy_(y)
        graph.replay()
        eager = ops.beam_select(live, at, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(result, eager))
        assert torch.equal(result[2].cpu(), plain.beam_select(x, y, 8)[2])


# ----------------------------------------------------------------------------------------------------------------------
# states that change places
# ----------------------------------------------------------------------------------------------------------------------
def check_reorder(ops, tensors, slots, parents, axis=0):
    want = plain.reorder_states(tensors, slots, parents, axis)
    live = [t.cuda() for t in tensors]
    ops.reorder_states(live, slots.cuda(), parents.cuda(), axis=axis)
    for got, expected in zip(live, want):
        assert torch.equal(got.cpu(), expected)


def random_rows(shape, dtype, g):
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g).to(dtype)
    return torch.randint(0, 100, shape, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32, torch.int32, torch.uint8, torch.int64])
@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 13, 16, 31, 33, 64])
@pytest.mark.parametrize("width", [1, 7, 64, 1025])
def test_reorder_widths(ops, dtype, beams, width):
    g = torch.Generator().manual_seed(width)
    slots = torch.randperm(3 * beams + 4, generator=g)[:3 * beams].view(3, beams).to(torch.int32)
    parents = torch.randint(0, beams, (3, beams), generator=g).to(torch.int32)
    check_reorder(ops, [random_rows((3 * beams + 4, width), dtype, g)], slots, parents)


@pytest.mark.parametrize("axis", [0, 1, 2])
def test_reorder_axes_and_rows_of_a_beam(ops, axis):
    g = torch.Generator().manual_seed(axis)
    shape = [3, 2, 5, 4]
    shape[axis] = 40
    slots = torch.randperm(40, generator=g)[:2 * 4 * 3].view(2, 4, 3).to(torch.int32)
    slots[0, 1, 2] = slots[1, 3, 0] = -1
    parents = torch.tensor([[1, 0, 3, 3], [2, 2, 2, 2]], dtype=torch.int32)
    check_reorder(ops, [random_rows(shape, F32, g), random_rows(shape, BF16, g)], slots, parents, axis)


def test_reorder_many_tensors_of_many_sizes(ops):
    g = torch.Generator().manual_seed(0)
    slots = torch.randperm(12, generator=g)[:8].view(2, 4).to(torch.int32)
    parents = torch.tensor([[3, 0, 1, 2], [0, 0, 1, 3]], dtype=torch.int32)
    tensors = [random_rows((12, 1 + 37 * i % 900), (F32, BF16, torch.int32)[i % 3], g) for i in range(70)] + [torch.zeros((12, 0)), torch.zeros((0, 3))]
    check_reorder(ops, tensors, slots, parents)


def test_reorder_leaves_alone_what_has_no_place(ops):
    """Rows and parents outside their range, unmoved beams, rows of nobody."""
    g = torch.Generator().manual_seed(0)
    slots = torch.tensor([[0, 1, 2, 3], [-1, 5, 99, 6]], dtype=torch.int32)
    parents = torch.tensor([[0, 7, -1, 1], [1, 0, 1, 2]], dtype=torch.int32)
    check_reorder(ops, [random_rows((9, 50), F32, g)], slots, parents)
    check_reorder(ops, [random_rows((9, 50), F32, g)], slots[:0], parents[:0])


@pytest.mark.parametrize("width", [64, 7])
def test_reorder_from_beams_that_take_over_nothing_themselves(ops, width):
    """A parent may have no parent of its own: its row goes to the others all the same, also where theirs is row 0."""
    g = torch.Generator().manual_seed(0)
    slots = torch.tensor([[0, 5, 3, 2], [6, 8, 7, 1]], dtype=torch.int32)
    for parents in ([[1, -1, 0, 99], [3, 3, -7, -1]], [[2, 2, -1, 2], [1, 4, 1, 1]], [[1, 99, 1, 1], [0, -1, 64, 65]]):
        check_reorder(ops, [random_rows((9, width), F32, g), random_rows((9, width), BF16, g)], slots, torch.tensor(parents, dtype=torch.int32))
        check_reorder(ops, [random_rows((9, width), F32, g)], slots.view(2, 2, 2).transpose(0, 1).contiguous(), torch.tensor(parents, dtype=torch.int32).view(2, 4)[:, :2].contiguous())


def test_reorder_large_rows(ops):
    """Offsets beyond 32 bits: rows of 96 MiB, seventy of them."""
    rows, width = 70, 24 << 20
    live = torch.empty((rows, width), dtype=F32, device="cuda")
    for r in range(rows):
        live[r] = torch.arange(width, device="cuda", dtype=F32) * (r + 1)
    slots = torch.tensor([[0, 69, 35, 68]], dtype=torch.int32).cuda()
    parents = torch.tensor([[1, 2, 3, 3]], dtype=torch.int32).cuda()
    ops.reorder_states([live], slots, parents)
    for row, source in ((0, 69), (69, 35), (35, 68), (68, 68), (1, 1), (67, 67)):
        assert torch.equal(live[row], torch.arange(width, device="cuda", dtype=F32) * (source + 1))


def test_reorder_captured(ops):
    g = torch.Generator().manual_seed(3)
    start = random_rows((10, 333), F32, g)
    live = start.cuda()
    slots, parents = torch.tensor([[1, 4, 7, 9]], dtype=torch.int32).cuda(), torch.tensor([[0, 1, 2, 3]], dtype=torch.int32).cuda()
    ops.reorder_states([live], slots, parents)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reorder_states([live], slots, parents)
    expected = start
    for step in ([1, 0, 0, 2], [3, 3, 1, 0], [2, 1, 0, 3]):
        parents.copy_(torch.tensor([step], dtype=torch.int32))
        expected = plain.reorder_states([expected], slots, parents)[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(live.cpu(), expected)


# ----------------------------------------------------------------------------------------------------------------------
# together
# ----------------------------------------------------------------------------------------------------------------------
def test_a_beam_search(ops):
    """Three prompts, four beams each, some steps: one attention over cached keys, a state beside it, a head.  Every step the attention reads the prompt once per
    request, the best continuations are chosen, and what the beams hold behind the prompt (a page and a state) moves with them.  The oracle keeps whole
    hypotheses and works each from its first token, in 64 bits."""
    g = torch.Generator().manual_seed(11)
    heads, kv_heads, dim, page, beams, steps, vocab = 4, 2, 32, 16, 4, 9, 997
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (37, 16, 70)]
    embed = torch.randn((vocab, heads * dim), generator=g, dtype=torch.float64)
    make_q, make_k, make_v = (torch.randn((heads * dim, n * dim), generator=g, dtype=torch.float64) * 0.08 for n in (heads, kv_heads, kv_heads))
    head = torch.randn((heads * dim, vocab), generator=g, dtype=torch.float64) * 0.15

    def oracle_logits(tokens):
        x = embed[tokens]
        q, k, v = (x[-1] @ make_q).view(heads, dim), (x @ make_k).view(-1, kv_heads, dim), (x @ make_v).view(-1, kv_heads, dim)
        out = torch.stack([torch.softmax(k[:, h // 2] @ q[h] * dim ** -0.5, 0) @ v[:, h // 2] for h in range(heads)]).view(-1)
        state = torch.zeros(heads * dim, dtype=torch.float64)
        for row in x:
            state = 0.5 * state + row
        return (out + state) @ head

    # the oracle
    found = []
    for prompt in prompts:
        live = [(0.0, [])]
        for _ in range(steps):
            every = []
            for score, tokens in live:
                chances = torch.log_softmax(oracle_logits(prompt + tokens), 0) + score
                values, at = chances.topk(beams)
                every += [(v, tokens + [t]) for v, t in zip(values.tolist(), at.tolist())]
            every.sort(key=lambda c: -c[0])
            assert every[beams - 1][0] - every[beams][0] > 1e-4 if len(every) > beams else True  # (the case says something)
            live = every[:beams]
        found.append(live)

    # the operators
    dev = "cuda"
    f32 = lambda t: t.to(F32).to(dev)  # noqa: E731
    tables_of, pages = [], 1
    whole = [len(p) // page for p in prompts]
    width = max(whole) + 2
    tables = torch.zeros((3 * beams, width), dtype=torch.int32)
    own_pages = torch.zeros((3, beams, 2), dtype=torch.int32)
    for r, n in enumerate(whole):
        for j in range(beams):
            tables[r * beams + j, :n] = torch.arange(pages, pages + n)
        pages += n
        for j in range(beams):
            own_pages[r, j] = torch.tensor([pages, pages + 1])
            tables[r * beams + j, n:n + 2] = own_pages[r, j]
            pages += 2
    k_cache, v_cache = torch.full((pages, kv_heads, page, dim), math.nan, device=dev), torch.full((pages, kv_heads, dim, page), math.nan, device=dev)
    state = torch.zeros((3 * beams + 1, heads * dim), device=dev)
    for r, prompt in enumerate(prompts):
        x = embed[prompt]
        k, v = (x @ make_k).view(-1, kv_heads, dim), (x @ make_v).view(-1, kv_heads, dim)
        s = torch.zeros(heads * dim, dtype=torch.float64)
        for row in x[:-1]:
            s = 0.5 * s + row
        for j in range(beams):
            state[r * beams + j] = f32(s)
            for n in range(len(prompt) - 1):
                at = tables[r * beams + j, n // page]
                k_cache[at, :, n % page], v_cache[at, :, :, n % page] = f32(k[n]), f32(v[n])
    tables = tables.to(dev)
    starts = torch.tensor([0, beams, 2 * beams, 3 * beams], dtype=torch.int32, device=dev)
    shared = torch.tensor([n * page for n in whole], dtype=torch.int32, device=dev)
    lens = torch.tensor([len(p) for p in prompts for _ in range(beams)], dtype=torch.int32, device=dev)
    shared = torch.minimum(shared, lens.view(3, beams)[:, 0] - 1).to(torch.int32)  # (the newest token's key is every beam's own)
    tokens = torch.tensor([p[-1] for p in prompts for _ in range(beams)], device=dev)
    scores = torch.full((3, beams), -math.inf, device=dev)
    scores[:, 0] = 0
    slots, workspace = torch.arange(3 * beams, dtype=torch.int32, device=dev).view(3, beams), Workspace(torch.device(dev))
    weights = [f32(t) for t in (embed, make_q, make_k, make_v, head)]
    rows = torch.arange(3 * beams, device=dev)
    histories = torch.zeros((3, beams, 0), dtype=torch.long, device=dev)
    own_pages = own_pages.to(dev)
    for _ in range(steps):
        x = weights[0][tokens]
        at = (lens - 1).long()
        where = tables[rows, at // page].long()
        k_cache[where, :, at % page] = (x @ weights[2]).view(-1, kv_heads, dim)
        v_cache[where, :, :, at % page] = (x @ weights[3]).view(-1, kv_heads, dim)
        state[rows] = 0.5 * state[rows] + x
        out = ops.shared_prefix_attention((x @ weights[1]).contiguous(), heads, kv_heads, dim, k_cache, v_cache, page, tables, lens, starts, shared, beams, width * page,
                                          dim ** -0.5, workspace)
        scores, parents, chosen = ops.beam_select(((out + state[rows]) @ weights[4]).contiguous(), scores, beams)
        ops.reorder_states([k_cache, v_cache], own_pages, parents)
        ops.reorder_states([state], slots, parents)
        histories = torch.cat([histories.gather(1, parents.long()[:, :, None].expand(-1, -1, histories.shape[2])), chosen.long()[:, :, None]], dim=2)
        tokens = chosen.view(-1).long()
        lens += 1
    for r in range(3):
        assert histories[r].tolist() == [tokens for _, tokens in found[r]]
        # a step's log-probability is off by float32 products of 128 terms; some 1e-5 each here, nine steps
        torch.testing.assert_close(scores[r].cpu().double(), torch.tensor([score for score, _ in found[r]], dtype=torch.float64), rtol=0, atol=2e-4)
