"""What the operators for several continuations of one prompt refuse, before anything is launched."""
import ctypes
import math
import random

import pytest
import torch

from velox_amd.kernels import build
from velox_amd.kernels.hip_ops import HipOps, KernelError


class _Nothing:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture()
def ops():
    """The checks alone: no library, so that anything that passes them says so."""
    made = object.__new__(HipOps)
    made.device = torch.device("cpu")
    made._index = -1
    made.num_cus = 256
    made._raw_stream = None
    made._shared_prefix = {dim: _Nothing() for dim in range(16, 272, 16)}
    made._beams = _Nothing()
    return made


class _Workspace:
    def get(self, name, numel):
        return torch.empty(numel)


def attention(**changed):
    a = dict(qkv=torch.zeros((3, 8 * 64)), num_heads=4, num_kv_heads=2, head_dim=64, k_cache=torch.zeros((9, 2, 16, 64)), v_cache=torch.zeros((9, 2, 64, 16)), block_size=16,
             block_tables=torch.zeros((3, 4), dtype=torch.int32), kv_lens=torch.ones(3, dtype=torch.int32), group_starts=torch.tensor([0, 3], dtype=torch.int32),
             shared_lens=torch.tensor([1], dtype=torch.int32), largest_group=3, max_kv_len=64, scale=0.125, workspace=_Workspace())
    a.update(changed)
    return a


@pytest.mark.parametrize("changed,says", [
    (dict(qkv=torch.zeros((3, 8 * 64), dtype=torch.float16)), "float32 or bfloat16"),
    (dict(qkv=torch.zeros((3, 8 * 64 + 1))), "rows of"),
    (dict(qkv=torch.zeros((4, 8 * 64))), "qkv"),
    (dict(qkv=torch.zeros((3, 16 * 64))[:, ::2]), "contiguous"),
    (dict(num_heads=5), "multiple"),
    (dict(num_kv_heads=0), "multiple"),
    (dict(head_dim=60), "head_dim"),
    (dict(head_dim=512), "head_dim"),
    (dict(k_cache=torch.zeros((9, 2, 16, 64), dtype=torch.bfloat16)), "k_cache"),
    (dict(k_cache=torch.zeros((0, 2, 16, 64))), "without pages"),
    (dict(v_cache=torch.zeros((9, 2, 16, 64))), "v_cache"),
    (dict(block_size=4), "block_size"),
    (dict(block_size=24), "block_size"),
    (dict(block_tables=torch.zeros((2, 4), dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros((3, 4), dtype=torch.int64)), "block_tables"),
    (dict(max_kv_len=65), "cannot cover"),
    (dict(max_kv_len=-1), "cannot cover"),
    (dict(kv_lens=torch.ones(3, dtype=torch.int64)), "kv_lens"),
    (dict(kv_lens=torch.ones((3, 1), dtype=torch.int32)), "kv_lens"),
    (dict(group_starts=torch.tensor([0, 1, 3], dtype=torch.int32)), "group_starts"),
    (dict(shared_lens=torch.tensor([[1]], dtype=torch.int32)), "shared_lens"),
    (dict(group_starts=torch.zeros(1026, dtype=torch.int32), shared_lens=torch.zeros(1025, dtype=torch.int32)), "at most 1024"),
    (dict(largest_group=0), "largest group"),
    (dict(largest_group=4), "largest group"),
    (dict(scale=0.0), "scale"),
    (dict(scale=math.nan), "scale"),
    (dict(scale=1e39), "scale"),
    (dict(block_size=131072), "block_size"),
    (dict(block_size=65536, block_tables=torch.zeros((3, 513), dtype=torch.int32), max_kv_len=2 ** 25 + 1), "at most 33554432"),
    (dict(sinks=torch.zeros(5)), "sinks"),
    (dict(sinks=torch.zeros(4, dtype=torch.bfloat16)), "sinks"),
    (dict(workspace=None), "workspace"),
])
def test_attention_refuses(ops, changed, says):
    with pytest.raises(KernelError, match=says):
        ops.shared_prefix_attention(**attention(**changed))


@pytest.mark.parametrize("num_seqs,longest", [(65536, 100), (65536, 1), (65535, 1 << 20), (1025, 1 << 25)])
def test_attention_refuses_more_than_it_counts(ops, num_seqs, longest):
    with pytest.raises(KernelError, match="more than one call takes"):
        ops._shared_prefix_shape(256, num_seqs, 1, 28, 4, 128, 2, 2, longest)


def test_attention_of_no_sequences(ops):
    out = ops.shared_prefix_attention(**attention(qkv=torch.zeros((0, 8 * 64)), block_tables=torch.zeros((0, 4), dtype=torch.int32), kv_lens=torch.zeros(0, dtype=torch.int32),
                                                  group_starts=torch.zeros(1, dtype=torch.int32), shared_lens=torch.zeros(0, dtype=torch.int32), largest_group=1))
    assert out.shape == (0, 256)


@pytest.mark.parametrize("heads,kv_heads,dim", [(28, 4, 128), (12, 2, 128), (32, 1, 64), (8, 8, 256), (3, 1, 16)])
def test_attention_items_are_enough(ops, heads, kv_heads, dim):
    """The bound on the items that the launch has room for, against the kernels' own count, over lengths and groups at random."""
    import random

    rng = random.Random(heads)
    group = heads // kv_heads
    for _ in range(300):
        sizes = [rng.choice([0, 1, 2, 3, 17, 70]) for _ in range(rng.randint(0, 9))]
        num_seqs = max(1, sum(sizes) + rng.randint(0, 5))
        element_size = rng.choice([2, 4])
        tile = 32 if element_size == 2 else 16
        row_tiles, target, items, rows = ops._shared_prefix_shape(256, num_seqs, len(sizes), heads, kv_heads, dim, element_size, max(sizes + [1]), rng.choice([1100, 40000]))
        own_blocks = -(-group // 16)
        shared_work, own_work = [], []  # (row blocks, steps) of the groups, tiles of the sequences
        for size in sizes:
            shared = rng.choice([0, 1, 5, 128, 1000, 33333]) if size > 1 else 0
            if shared:
                shared_work.append((-(-size * group // (16 * row_tiles)), -(-shared // (64 if row_tiles == 8 else 4 * tile))))
            for _ in range(size):
                more = rng.choice([0, 1, 200, 5000])
                own_work.append(-(-(shared + more - shared // tile * tile) // tile) if more else 0)
        own_work += [-(-rng.choice([0, 1, 200, 5000]) // tile) for _ in range(num_seqs - len(own_work))]
        per = max(1, -(-(sum(x * y for x, y in shared_work) + -(-own_blocks * sum(own_work) // 4)) // target))
        if per == 2 and row_tiles != 8:
            per = rng.choice([1, 2])  # (which one goes by the longest group)
        shared_items = sum(x * -(-y // per) for x, y in shared_work)
        own_items = sum(own_blocks * max(1, -(-y // per)) for y in own_work)
        assert shared_items + -(-own_items // 4) <= items
        assert shared_items * 16 * row_tiles + own_items * 16 <= rows


class _Asked(Exception):
    pass


class _Recording:
    """Says how many elements a call asks for, and ends it."""

    def get(self, name, numel):
        raise _Asked(numel)


def scratch_of_a_call(ops, heads, kv_heads, dim, dtype, num_seqs, num_groups, largest, longest):
    """Elements that a call of these sizes asks its workspace for."""
    page = 16
    call = attention(
        qkv=torch.empty((num_seqs, heads * dim), dtype=dtype), num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, k_cache=torch.empty((1, kv_heads, page, dim), dtype=dtype),
        v_cache=torch.empty((1, kv_heads, dim, page), dtype=dtype), block_size=page, block_tables=torch.empty((num_seqs, -(-longest // page)), dtype=torch.int32),
        kv_lens=torch.empty(num_seqs, dtype=torch.int32), group_starts=torch.empty(num_groups + 1, dtype=torch.int32), shared_lens=torch.empty(num_groups, dtype=torch.int32),
        largest_group=largest, max_kv_len=longest, workspace=_Recording())
    try:
        ops.shared_prefix_attention(**call)
    except _Asked as asked:
        return asked.args[0]
    except AssertionError:
        return 0  # (the launch was reached: nothing was asked for)


@pytest.mark.parametrize("heads,kv_heads,dim,num_seqs,num_groups,longest", [
    (12, 2, 128, 81, 1, 32768), (8, 1, 128, 65, 1, 32768), (14, 2, 64, 124, 1, 1000), (12, 2, 128, 210, 1, 1000), (5, 1, 80, 99, 1, 5000),
])
def test_attention_scratch_of_large_float32_groups(ops, heads, kv_heads, dim, num_seqs, num_groups, longest):
    """Single row tiles, two workgroups to a compute unit, items written down ahead."""
    assert 0 < scratch_of_a_call(ops, heads, kv_heads, dim, torch.float32, num_seqs, num_groups, num_seqs, longest) <= ops.shared_prefix_scratch_elems(heads, kv_heads, dim, num_seqs, num_groups)


@pytest.mark.parametrize("num_cus", [256, 64, 304])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 2, 128), (28, 4, 64), (8, 1, 128), (40, 8, 128), (5, 1, 80), (34, 2, 32), (3, 1, 256), (32, 32, 64), (600, 300, 16)])
def test_attention_scratch_of_any_call_within_limits(ops, heads, kv_heads, dim, num_cus):
    rng, ops.num_cus, shared_out = random.Random(heads + num_cus), num_cus, 0
    for _ in range(60):
        most_seqs, most_groups = rng.choice([1, 5, 40, 64, 65, 130, 300]), rng.choice([0, 1, 6, 64, 65, 200])
        most = ops.shared_prefix_scratch_elems(heads, kv_heads, dim, most_seqs, most_groups)
        for _ in range(4):
            num_seqs, num_groups = rng.choice([most_seqs, rng.randint(1, most_seqs)]), rng.choice([most_groups, rng.randint(0, most_groups)])
            asked = scratch_of_a_call(ops, heads, kv_heads, dim, rng.choice([torch.float32, torch.float32, torch.bfloat16]), num_seqs, num_groups,
                                      rng.choice([num_seqs, rng.randint(1, num_seqs)]), rng.choice([90, 1000, 5000, 32768]))
            assert asked <= most
            shared_out += asked > 0
    assert shared_out > 60


def test_kernels_and_checks_have_the_same_limits(ops):
    """Also what a call may leave behind, which both sides count."""
    ops._beams, ops._shared_prefix = None, {}
    assert ops.beam_library() is not None  # (a library with other limits is refused)
    lib = ops.shared_prefix_library(64)
    count, elems = lib.velox_shared_prefix_room, (ctypes.c_longlong * 2)()
    count.argtypes, count.restype = [ctypes.c_int] * 6 + [ctypes.c_void_p] * 2, None
    rng = random.Random(3)
    for _ in range(500):
        num_seqs, num_groups, group = rng.randint(1, 3000), rng.choice([0, 1, rng.randint(0, 1024)]), rng.choice([1, 2, 7, 16, 17, 64])
        sizes = num_seqs, num_groups, group, rng.choice([1, 2, 8]), rng.choice([1, 32, 64, 512]), rng.randint(1, num_seqs)
        count(*sizes, ctypes.addressof(elems), ctypes.addressof(elems) + 8)
        assert tuple(elems) == ops._shared_prefix_room(*sizes)


@pytest.mark.parametrize("changed", ["MAX_BEAMS", "MAX_KEPT", "MAX_BEAM_VOCAB", "MAX_MOVED", "MAX_MOVED_TENSORS", "MAX_PREFIX_GROUPS", "MAX_PREFIX_KEYS"])
def test_a_library_of_other_limits_is_refused(ops, changed):
    ops._beams, ops._shared_prefix = None, {}
    setattr(ops, changed, getattr(ops, changed) + 1)
    with pytest.raises(KernelError, match="other limits"):
        ops.shared_prefix_library(64) if "PREFIX" in changed else ops.beam_library()


@pytest.mark.parametrize("logits,scores,keep,says", [
    (torch.zeros((4, 9), dtype=torch.bfloat16), torch.zeros((2, 2)), 4, "logits"),
    (torch.zeros((4, 9)).double(), torch.zeros((2, 2)), 4, "logits"),
    (torch.zeros((4, 18))[:, ::2], torch.zeros((2, 2)), 4, "contiguous"),
    (torch.zeros((4, 9)), torch.zeros((2, 2)).double(), 4, "scores"),
    (torch.zeros((4, 9)), torch.zeros((2, 3)), 4, "do not go"),
    (torch.zeros((4, 9)), torch.zeros(4), 4, "do not go"),
    (torch.zeros((4, 9)), torch.zeros((2, 2)), 0, "keep"),
    (torch.zeros((4, 9)), torch.zeros((2, 2)), 19, "keep"),
    (torch.zeros((4, 99)), torch.zeros((2, 2)), 65, "keep"),
    (torch.zeros((257, 9)), torch.zeros((1, 257)), 4, "beams"),
    (torch.zeros((4, 0)), torch.zeros((2, 2)), 1, "tokens"),
    (torch.zeros((0, 9)), torch.zeros((2, 0)), 1, "beams"),
    (torch.zeros((65536, 1)), torch.zeros((65536, 1)), 1, "grid"),
])
def test_selection_refuses(ops, logits, scores, keep, says):
    with pytest.raises(KernelError, match=says):
        ops.beam_select(logits, scores, keep)


def test_selection_of_no_requests(ops):
    values, parents, tokens = ops.beam_select(torch.zeros((0, 9)), torch.zeros((0, 2)), 4)
    assert values.shape == parents.shape == tokens.shape == (0, 4) and parents.dtype == tokens.dtype == torch.int32


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("tensors,slots,parents,axis,says", [
    ([torch.zeros((9, 4))], ints([0, 1]).long(), ints([0, 1]), 0, "slots"),
    ([torch.zeros((9, 4))], ints([0, 1]), ints([0, 1]).long(), 0, "parents"),
    ([torch.zeros((9, 4))], ints([0, 1]), ints([0, 1, 2]), 0, "do not go"),
    ([torch.zeros((9, 4))], ints(0, 1), ints(0, 1), 0, "do not go"),
    ([torch.zeros((9, 4))], torch.zeros((1, 65), dtype=torch.int32), torch.zeros((1, 65), dtype=torch.int32), 0, "beams"),
    ([torch.zeros((9, 4))], torch.zeros((1, 2, 65536), dtype=torch.int32), ints([0, 1]), 0, "rows"),
    ([torch.zeros((9, 4))], ints([0, 1]), ints([0, 1]), 2, "dimension"),
    ([torch.zeros((9, 4))], ints([0, 1]), ints([0, 1]), -1, "dimension"),
    ([torch.zeros((9, 8))[:, ::2]], ints([0, 1]), ints([0, 1]), 0, "contiguous"),
    ([torch.zeros((65536, 9, 1))], ints([0, 1]), ints([0, 1]), 1, "grid"),
])
def test_reorder_refuses(ops, tensors, slots, parents, axis, says):
    with pytest.raises(KernelError, match=says):
        ops.reorder_states(tensors, slots, parents, axis=axis)


def test_reorder_refuses_shared_memory(ops):
    t = torch.zeros((9, 4))
    for pair in ([t, t], [t, t[3:]], [t[:5], t[4:]]):
        with pytest.raises(KernelError, match="share memory"):
            ops.reorder_states(pair, ints([0, 1]), ints([0, 1]))


def test_reorder_of_nothing(ops):
    ops.reorder_states([], ints([0, 1]), ints([1, 0]))
    ops.reorder_states([torch.zeros((9, 0))], ints([0, 1]), ints([1, 0]))
    ops.reorder_states([torch.zeros((9, 4))], torch.zeros((0, 2), dtype=torch.int32), torch.zeros((0, 2), dtype=torch.int32))
