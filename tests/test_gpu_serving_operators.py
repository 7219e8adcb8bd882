"""The serving operators on device pointers (hf_cuda_attention_packed, hf_cuda_attention_tree, hf_cuda_pages_*) against plain
64-bit implementations (serving_reference.py): types, head layouts, lengths around the page and tile borders, strided
views, empty sequences, garbage outside the rows in use, captured graphs, and a serving run of all of them together."""
import math
import threading

import pytest

import serving_reference as ref
from huggingfaceeacp_b200 import native

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PAGE = native.PAGE_ROWS
TYPES = ["f32", "bf16", "f16"]


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    native.operators_sync(0, _stream())


HEADS = [(8, 1, 256), (8, 2, 128), (4, 4, 64), (6, 2, 96), (7, 1, 80), (3, 3, 8), (10, 2, 40), (2, 2, 200)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _offsets(lengths, begin=0):
    at = [begin]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _fused(g, rows, heads, kv_heads, width, dtype):
    """q, k, v as views of one [rows, q | k | v] buffer, and its row stride."""
    qkv = _normal(g, rows, (heads + 2 * kv_heads) * width, dtype=dtype)
    parts = qkv.split([heads * width, kv_heads * width, kv_heads * width], 1)
    return [x.unflatten(1, (-1, width)) for x in parts], qkv.stride(0)


def _room(size):
    return torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")


def _run_packed(code, q, k, v, out, lengths, stride, scale=None, begin=0, stream=None):
    heads, width = q.shape[1:]
    plan = native.PackedAttention(code, heads, k.shape[1], width, scale=scale)
    offsets = _ints(_offsets(lengths, begin))
    room = _room(plan.workspace_bytes(len(lengths), len(q)))
    plan.run(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), len(lengths), len(q),
             q_stride=stride, k_stride=stride, v_stride=stride, workspace=room.data_ptr(), workspace_bytes=room.numel(),
             stream=_stream() if stream is None else stream)
    return offsets, room


# ---- packed prompts ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_packed_prompts_of_every_layout(kind, heads):
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    lengths = [1, 0, 130, 17, 64, 3]
    g = torch.Generator("cuda").manual_seed(1)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    ref.close(out, expected, size, q, k, d ** -0.5, max(lengths))


@pytest.mark.parametrize("lengths", [[1], [2], [15], [16], [63], [65], [127], [128], [129], [191, 193], [257], [500, 1, 300]],
                         ids=str)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(8, 1, 256), (8, 2, 128), (2, 2, 64)], ids=str)
def test_packed_prompts_around_the_tile_borders(kind, lengths, heads):
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    g = torch.Generator("cuda").manual_seed(2)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride, scale=0.11)
    expected, size = ref.packed(q, k, v, lengths, 0.11)
    ref.close(out, expected, size, q, k, 0.11, max(lengths))


@pytest.mark.parametrize("kind", TYPES)
def test_packed_prompts_of_many_sequences(kind):
    code, dtype = ref.TYPES[kind]
    lengths = [(i * 37) % 23 for i in range(150)]
    g = torch.Generator("cuda").manual_seed(3)
    (q, k, v), stride = _fused(g, sum(lengths), 4, 2, 64, dtype)
    out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, 64 ** -0.5)
    ref.close(out, expected, size, q, k, 64 ** -0.5, max(lengths))


@pytest.mark.parametrize("heads", [(16, 4, 128), (12, 12, 64)], ids=str)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lengths", [[i * 37 % 41 for i in range(300)], [95, 97] * 20, [700, 400, 1, 0, 1300, 650]],
                         ids=["short", "between", "long"])
def test_packed_prompts_that_fill_every_sm(kind, heads, lengths):
    """Enough rows for two query tiles a CTA, taken where the prompts are long, or one where they are short."""
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    g = torch.Generator("cuda").manual_seed(31)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    ref.close(out, expected, size, q, k, d ** -0.5, max(lengths))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(8, 1, 256), (4, 2, 128), (5, 5, 72)], ids=str)
def test_packed_rows_outside_every_sequence_are_left_alone(kind, heads):
    """Rows before the first and behind the last sequence hold NaN and infinities: neither read nor written."""
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    lengths, before, behind = [70, 9], 5, 77
    g = torch.Generator("cuda").manual_seed(4)
    (q, k, v), stride = _fused(g, before + sum(lengths) + behind, h, kv, d, dtype)
    for x in (q, k, v):
        x[:before] = math.inf
        x[before + sum(lengths):] = math.nan
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride, begin=before)
    used = slice(before, before + sum(lengths))
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5, begin=before)
    ref.close(out[used], expected[used], size[used], q[used], k[used], d ** -0.5, max(lengths))
    assert bool((out[:before] == 7.0).all()) and bool((out[before + sum(lengths):] == 7.0).all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_packed_garbage_reaches_only_the_rows_that_attend_to_it(kind, value):
    code, dtype = ref.TYPES[kind]
    lengths, h, kv, d, bad = [90, 40], 8, 2, 128, 60
    g = torch.Generator("cuda").manual_seed(5)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    clean = [x.clone() for x in (q, k, v)]
    v[bad, :, 3] = value
    k[bad, 0, 1] = math.nan  # kv head 0: the whole row of its query heads
    out = torch.empty(q.shape, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(*clean, lengths, d ** -0.5)
    fine = torch.ones(sum(lengths), h, d, dtype=torch.bool, device="cuda")
    fine[bad:lengths[0], :, 3] = False
    fine[bad:lengths[0], : h // kv] = False
    where = fine.nonzero(as_tuple=True)
    tol = ref.tolerance(expected, size, *clean[:2], d ** -0.5, max(lengths), dtype)
    assert bool(((out.double() - expected).abs() <= tol)[where].all())
    assert bool(torch.isnan(out[bad:lengths[0], : h // kv]).all())
    got = out[bad:lengths[0], h // kv:, 3].float()
    assert bool((torch.isnan(got) if math.isnan(value) else got == value).all())


@pytest.mark.parametrize("kind", TYPES)
def test_packed_scores_far_apart(kind):
    """Large scores: the running maximum rises from tile to tile, and weights underflow to zero."""
    code, dtype = ref.TYPES[kind]
    lengths, d = [400], 64
    g = torch.Generator("cuda").manual_seed(6)
    (q, k, v), stride = _fused(g, 400, 4, 2, d, dtype)
    k *= (torch.arange(400, device="cuda") / 40.0).to(dtype)[:, None, None]
    q *= 2
    out = torch.empty(q.shape, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    ref.close(out, expected, size, q, k, d ** -0.5, 400)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 3e4, 1e-6])
def test_packed_fp32_keeps_its_digits_at_any_magnitude(scale):
    """Rows of very different size, in one tile too: the relative error stays that of fp32."""
    lengths, d = [300], 256
    g = torch.Generator("cuda").manual_seed(7)
    (q, k, v), stride = _fused(g, 300, 8, 1, d, torch.float32)
    v *= scale
    k *= 10.0 ** (torch.arange(300, device="cuda") % 5 - 3)[:, None, None]
    out = torch.empty(q.shape, device="cuda")
    _run_packed(native.F32, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    ref.close(out, expected, size, q, k, d ** -0.5, 300)


# ---- trees ---------------------------------------------------------------------------------------------------------


class Cache:
    def __init__(self, kind, layers, pages, kv_heads, width, lengths, stride, seed, table=None):
        code, dtype = ref.TYPES[kind]
        g = torch.Generator("cuda").manual_seed(seed)
        self.keys = _normal(g, layers, pages, PAGE, kv_heads * width, dtype=dtype)
        self.values = _normal(g, layers, pages, PAGE, kv_heads * width, dtype=dtype)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        if table is None:
            table, at = [], 0
            for n in lengths:
                held = -(-n // PAGE)
                table.append(order[at : at + held] + [-1] * (stride - held))
                at += held
        refs = [sum(row[: -(-max(n, 0) // PAGE)].count(p) for row, n in zip(table, lengths)) for p in range(pages)]
        self.shape = (pages, PAGE, kv_heads, width)
        self.table, self.lengths, self.refs = _ints(table), _ints(lengths), _ints(refs)
        self.native = native.PageCache(code, layers, pages, kv_heads * width, len(lengths), stride, self.keys.data_ptr(),
                                       self.values.data_ptr(), self.table.data_ptr(), self.lengths.data_ptr(),
                                       self.refs.data_ptr())
        self.room = _room(self.native.workspace_bytes)
        self.result = _ints([-9, -9, -9])
        self.kind, self.code, self.dtype = kind, code, dtype

    def kw(self):
        return {"workspace": self.room.data_ptr(), "workspace_bytes": self.room.numel(), "stream": _stream()}

    def book(self):
        return ref.Book(self.keys, self.values, self.table.tolist(), self.lengths.tolist(), self.refs.tolist())

    def same(self, book):
        assert self.table.tolist() == book.table
        assert self.lengths.tolist() == book.lengths
        assert self.refs.tolist() == book.refs
        for got, want in ((self.keys, book.keys), (self.values, book.values)):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def _tree(cache, layer, heads, kv_heads, width, nodes, parents, seed, max_length, max_nodes=None, poison=False):
    g = torch.Generator("cuda").manual_seed(seed)
    (q, k, v), stride = _fused(g, sum(nodes) + 2, heads, kv_heads, width, cache.dtype)
    if poison:
        for x in (q, k, v):
            x[sum(nodes):] = math.nan
    out = torch.full(q.shape, 7.0, dtype=cache.dtype, device="cuda")
    plan = native.TreeAttention(cache.code, heads, kv_heads, width)
    offsets, up = _ints(_offsets(nodes)), _ints([p for row in parents for p in row] + [-1, -1])
    most = max_nodes or max(1, max(nodes))
    room = _room(plan.workspace_bytes(len(nodes), len(q), most, max_length))
    plan.run(cache.native, layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(),
             len(q), most, max_length, q_stride=stride, k_stride=stride, v_stride=stride, workspace=room.data_ptr(),
             workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.tree(q, k, v, nodes, parents, cache.keys[layer].view(cache.shape), cache.values[layer].view(cache.shape),
                              cache.table.tolist(), cache.lengths.tolist(), width ** -0.5)
    n = sum(nodes)
    if n:
        keys = max(cache.lengths.tolist()) + 64
        everything = torch.cat([k[:n], cache.keys[layer].view(-1, kv_heads, width)])
        ref.close(out[:n], expected[:n], size[:n], q[:n], everything, width ** -0.5, keys)
    assert bool((out[n:] == 7.0).all())


def _branching(n, seed):
    """Parents of a random tree of n nodes, several of them following the cache."""
    g = torch.Generator().manual_seed(seed)
    return [-1 if i == 0 else int(torch.randint(-1, i, (1,), generator=g)) for i in range(n)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_trees_of_every_layout(kind, heads):
    h, kv, d = heads
    lengths, nodes = [0, 1, 63, 64, 65, 200, 5], [3, 1, 0, 12, 7, 1, 20]
    cache = Cache(kind, 2, 20, kv, d, lengths, 5, 11)
    parents = [_branching(n, i) for i, n in enumerate(nodes)]
    _tree(cache, 1, h, kv, d, nodes, parents, 12, 200)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(8, 1, 256), (8, 2, 128), (16, 8, 64)], ids=str)
@pytest.mark.parametrize("lengths", [[0, 0], [1, 64], [700, 130], [4097, 3]], ids=str)
@pytest.mark.parametrize("nodes", [[1, 1], [64, 33], [0, 16]], ids=str)
def test_trees_of_one_to_64_nodes(kind, heads, lengths, nodes):
    h, kv, d = heads
    cache = Cache(kind, 1, 80, kv, d, lengths, 66, 13)
    _tree(cache, 0, h, kv, d, nodes, [_branching(n, 20 + i) for i, n in enumerate(nodes)], 14, max(lengths))


@pytest.mark.parametrize("kind", TYPES)
def test_decode_steps_of_many_sequences(kind):
    lengths = [(i * 97) % 300 for i in range(40)]
    cache = Cache(kind, 1, 260, 2, 128, lengths, 6, 15)
    _tree(cache, 0, 8, 2, 128, [1] * 40, [[-1]] * 40, 16, 300)


@pytest.mark.parametrize("heads", [(4, 1, 256), (6, 2, 40), (3, 3, 128)], ids=str)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths", [[1], [5, 0, 1, 9], [0, 0], [2] * 12], ids=str)
def test_packed_calls_of_a_few_rows(kind, heads, lengths):
    """The smallest calls; rows before and behind the prompts hold NaN and are left alone."""
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    before, used = 2, sum(lengths)
    g = torch.Generator("cuda").manual_seed(34)
    (q, k, v), stride = _fused(g, before + used + 3, h, kv, d, dtype)
    for x in (q, k, v):
        x[:before] = math.nan
        x[before + used:] = math.nan
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride, begin=before)
    rows = slice(before, before + used)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5, begin=before)
    if used:
        ref.close(out[rows], expected[rows], size[rows], q[rows], k[rows], d ** -0.5, max(lengths))
    assert bool((out[:before] == 7.0).all()) and bool((out[before + used:] == 7.0).all())


@pytest.mark.parametrize("heads", [(4, 1, 256), (6, 2, 40), (3, 3, 128)], ids=str)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,nodes", [([0], [1]), ([47], [1]), ([70, 0, 1, 64], [3, 1, 0, 7]), ([90, 65, 3] * 5, [1] * 15)],
                         ids=str)
def test_tree_calls_of_a_few_rows(kind, heads, lengths, nodes):
    """The smallest calls; page rows past a length, free pages and rows behind the last sequence hold NaN."""
    h, kv, d = heads
    pages = sum((n + PAGE - 1) // PAGE for n in lengths) + 2
    cache = Cache(kind, 1, pages, kv, d, lengths, 2, 35)
    for pool in (cache.keys, cache.values):
        held = torch.zeros(pages, PAGE, dtype=torch.bool)
        for row, n in zip(cache.table.tolist(), lengths):
            for j in range(n):
                held[row[j // PAGE], j % PAGE] = True
        pool[0][~held.cuda()] = math.nan
    _tree(cache, 0, h, kv, d, nodes, [_branching(n, n) for n in nodes], 36, max(lengths), poison=True)


@pytest.mark.parametrize("nodes", [1, 5])
@pytest.mark.parametrize("sequences", [38, 39, 41, 56, 67, 75, 113])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_trees_cut_at_every_place(kind, sequences, nodes):
    """One long cache among short and empty ones: CTAs begin and end on every tile of a sequence and before its first."""
    lengths = [(i * 61) % 131 for i in range(sequences)]
    lengths[sequences // 3] = 4000
    cache = Cache(kind, 1, sum((n + PAGE - 1) // PAGE for n in lengths) + 3, 4, 64, lengths, 63, 32)
    _tree(cache, 0, 8, 4, 64, [nodes] * sequences, [_branching(nodes, 2)] * sequences, 33, 4000)


@pytest.mark.parametrize("kind", TYPES)
def test_tree_garbage_in_the_cache_is_not_read(kind):
    """Page rows past a length, free pages, and drafted rows behind the last sequence hold NaN."""
    lengths = [70, 1, 129]
    cache = Cache(kind, 1, 12, 2, 64, lengths, 4, 17)
    for pool in (cache.keys, cache.values):
        held = torch.zeros(12, PAGE, dtype=torch.bool)
        for row, n in zip(cache.table.tolist(), lengths):
            for j in range(n):
                held[row[j // PAGE], j % PAGE] = True
        pool[0][~held.cuda()] = math.nan
    _tree(cache, 0, 8, 2, 64, [5, 1, 9], [_branching(n, n) for n in (5, 1, 9)], 18, 129, poison=True)


@pytest.mark.parametrize("kind", TYPES)
def test_tree_siblings_do_not_reach_each_other(kind):
    """A sibling's value of NaN or infinity stays with its own descendants."""
    code, dtype = ref.TYPES[kind]
    lengths, parents, h, kv, d = [100], [-1, 0, 0, 1, 2, 2], 4, 1, 128
    cache = Cache(kind, 1, 3, kv, d, lengths, 2, 19)
    g = torch.Generator("cuda").manual_seed(20)
    q, k, v = (_normal(g, 6, n, d, dtype=dtype) for n in (h, kv, kv))
    v[1], v[2] = math.inf, math.nan
    out = torch.empty_like(q)
    plan = native.TreeAttention(code, h, kv, d)
    offsets, up = _ints([0, 6]), _ints(parents)
    room = _room(plan.workspace_bytes(1, 6, 6, 100))
    plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(), 6, 6,
             100, workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.tree(q, k, v, [6], [parents], cache.keys[0].view(cache.shape), cache.values[0].view(cache.shape),
                              cache.table.tolist(), lengths, d ** -0.5)
    ref.close(out[:1], expected[:1], size[:1], q, k, d ** -0.5, 200)
    assert bool((out[[1, 3]] == math.inf).all()) and bool(torch.isnan(out[[2, 4, 5]]).all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 128, 200, 257, 1000])
def test_tree_infinities_wherever_the_keys_are_cut(kind, length):
    """Infinite values in the cache's first and last position and in one node: rows are exact in every other channel, for
    caches whose tiles fall differently on the CTAs."""
    code, dtype = ref.TYPES[kind]
    parents, h, kv, d = [-1, 0, 0, 1], 4, 2, 64
    cache = Cache(kind, 1, 18, kv, d, [length, 70], 17, 24)
    at = cache.table.tolist()[0]
    for j, channel in ((0, 5), (length - 1, 9)):
        if 0 <= j < length:
            cache.values[0, at[j // PAGE], j % PAGE, channel] = math.inf
    g = torch.Generator("cuda").manual_seed(25)
    q, k, v = (_normal(g, 8, n, d, dtype=dtype) for n in (h, kv, kv))
    v[2, 0, 11] = -math.inf
    out = torch.empty_like(q)
    plan = native.TreeAttention(code, h, kv, d)
    offsets, up = _ints([0, 4, 8]), _ints(parents * 2)
    room = _room(plan.workspace_bytes(2, 8, 4, 1000))
    plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(), 8, 4,
             1000, workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.tree(q, k, v, [4, 4], [parents] * 2, cache.keys[0].view(cache.shape), cache.values[0].view(cache.shape),
                              cache.table.tolist(), [length, 70], d ** -0.5)
    fine = torch.isfinite(expected)
    assert torch.equal(torch.isfinite(out), fine)
    tol = ref.tolerance(expected.nan_to_num(0, 0, 0), size.nan_to_num(0, 0, 0), q, cache.keys[0].view(-1, kv, d), d ** -0.5,
                        length + 8, dtype)
    assert bool(((out.double() - expected).abs() <= tol)[fine].all())
    assert bool((out.double()[~fine] == expected[~fine]).all())


@pytest.mark.parametrize("kind", TYPES)
def test_tree_pages_that_are_not_there_and_bounds(kind):
    """Page ids outside the pool are not attended; lengths and node counts are bounded by the call's."""
    lengths = [200, 130]
    cache = Cache(kind, 1, 6, 1, 64, lengths, 4, 21, table=[[2, -1, 5, 77777], [-5, 0, 6, -1]])
    _tree(cache, 0, 4, 1, 64, [3, 4], [[-1, 0, 1], [-1, -1, 1, 5]], 22, 200)
    # Both sequences have more positions than max_length, the second more nodes than max_nodes.
    g = torch.Generator("cuda").manual_seed(23)
    (q, k, v), stride = _fused(g, 7, 4, 1, 64, cache.dtype)
    out = torch.full(q.shape, 7.0, dtype=cache.dtype, device="cuda")
    plan, offsets, up = native.TreeAttention(cache.code, 4, 1, 64), _ints([0, 2, 7]), _ints([-1, 0, -1, 0, 1, 2, 3])
    room = _room(plan.workspace_bytes(2, 7, 3, 100))
    plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(), 7, 3,
             100, q_stride=stride, k_stride=stride, v_stride=stride, workspace=room.data_ptr(), workspace_bytes=room.numel(),
             stream=_stream())
    expected, size = ref.tree(q[:5], k[:5], v[:5], [2, 3], [[-1, 0], [-1, 0, 1]], cache.keys[0].view(cache.shape),
                              cache.values[0].view(cache.shape), cache.table.tolist(), [100, 100], 64 ** -0.5)
    ref.close(out[:5], expected, size, q[:5], cache.keys[0].view(-1, 1, 64), 64 ** -0.5, 200)
    assert bool((out[5:] == 7.0).all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bound", [60, 109, 110, 150])
def test_tree_bounds_in_short_and_long_calls(kind, bound):
    """The call's bounds and missing pages on both sides of 112 keys, where the kernels change."""
    cache = Cache(kind, 1, 6, 1, 64, [200, 180], 4, 37, table=[[2, -1, 5, 77777], [-5, 0, 1, -1]])
    g = torch.Generator("cuda").manual_seed(38)
    (q, k, v), stride = _fused(g, 7, 4, 1, 64, cache.dtype)
    out = torch.full(q.shape, 7.0, dtype=cache.dtype, device="cuda")
    plan, offsets, up = native.TreeAttention(cache.code, 4, 1, 64), _ints([0, 2, 7]), _ints([-1, 0, -1, 0, 1, 2, 3])
    room = _room(plan.workspace_bytes(2, 7, 3, bound))
    plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(), 7, 3,
             bound, q_stride=stride, k_stride=stride, v_stride=stride, workspace=room.data_ptr(),
             workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.tree(q[:5], k[:5], v[:5], [2, 3], [[-1, 0], [-1, 0, 1]], cache.keys[0].view(cache.shape),
                              cache.values[0].view(cache.shape), cache.table.tolist(), [bound, bound], 64 ** -0.5)
    everything = torch.cat([k[:5], cache.keys[0].view(-1, 1, 64)])
    ref.close(out[:5], expected, size, q[:5], everything, 64 ** -0.5, bound + 3)
    assert bool((out[5:] == 7.0).all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("length", [10, 128, 300])
def test_tree_siblings_in_short_and_long_calls(kind, length):
    """A sibling's value of NaN or infinity stays with its own descendants, over caches of either kernel."""
    code, dtype = ref.TYPES[kind]
    parents, h, kv, d = [-1, 0, 0, 1, 2, 2], 4, 1, 128
    cache = Cache(kind, 1, 6, kv, d, [length], 5, 39)
    g = torch.Generator("cuda").manual_seed(40)
    q, k, v = (_normal(g, 6, n, d, dtype=dtype) for n in (h, kv, kv))
    v[1], v[2] = math.inf, math.nan
    out = torch.empty_like(q)
    plan = native.TreeAttention(code, h, kv, d)
    offsets, up = _ints([0, 6]), _ints(parents)
    room = _room(plan.workspace_bytes(1, 6, 6, length))
    plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(), 6, 6,
             length, workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.tree(q, k, v, [6], [parents], cache.keys[0].view(cache.shape), cache.values[0].view(cache.shape),
                              cache.table.tolist(), [length], d ** -0.5)
    everything = torch.cat([k, cache.keys[0].view(-1, kv, d)])
    ref.close(out[:1], expected[:1], size[:1], q, everything, d ** -0.5, length + 6)
    assert bool((out[[1, 3]] == math.inf).all()) and bool(torch.isnan(out[[2, 4, 5]]).all())


# ---- the cache's steps ---------------------------------------------------------------------------------------------


def _update(cache, release=(), forks=(), grow=None):
    book = cache.book()
    expected = book.update(release, forks, grow)
    lists = [_ints(list(release)), _ints([x for pair in forks for x in pair]), None if grow is None else _ints(grow)]
    cache.native.update(cache.result.data_ptr(), release=lists[0].data_ptr() if release else 0, releases=len(release),
                        forks=lists[1].data_ptr() if forks else 0, fork_count=len(forks),
                        grow=0 if grow is None else lists[2].data_ptr(), **cache.kw())
    assert cache.result.tolist() == expected
    cache.same(book)


@pytest.mark.parametrize("kind", TYPES)
def test_update_releases_forks_and_grows(kind):
    cache = Cache(kind, 3, 30, 2, 40, [100, 64, 0, 5, 130, 0, 0, 63], 4, 31)
    _update(cache, grow=[1, 1, 1, 1, 1, 0, 0, 1])
    _update(cache, release=[4, 4, -1, 99, 3], forks=[(0, 5), (7, 6), (0, 5), (1, 4), (0, 1), (2, 2), (0, -1), (88, 3)])
    _update(cache, grow=[1, 3, 0, 70, 0, 2, 65, 1])
    _update(cache, release=[0], forks=[(5, 0), (5, 3), (6, 2)], grow=[1, 0, 2, 3, -4, 1, 1, 0])
    _update(cache)


def test_update_copies_a_shared_page_for_all_but_the_last_that_grows():
    cache = Cache("f32", 2, 12, 1, 32, [70, 0, 0, 0], 3, 32)
    _update(cache, forks=[(0, 1), (0, 2), (0, 3)], grow=[1, 1, 1, 1])
    assert sorted(cache.refs.tolist(), reverse=True)[:6] == [4, 1, 1, 1, 1, 0]


def test_update_that_does_not_fit_grows_nothing():
    cache = Cache("bf16", 1, 6, 1, 64, [64, 128, 10], 3, 33)
    _update(cache, grow=[1, 60, 200])   # four pages wanted, two free
    _update(cache, grow=[1, 65, 1])     # the second would pass its row of three pages
    _update(cache, release=[1], grow=[1, 64, 100])


def test_update_of_many_sequences_and_pages():
    n = 1500
    lengths = [(i * 53) % 200 if i % 3 else 0 for i in range(n)]
    cache = Cache("f16", 1, 9000, 1, 8, lengths, 5, 34)
    _update(cache, release=list(range(0, n, 7)), forks=[(i + 1, i) for i in range(0, n - 1, 3)],
            grow=[i % 3 for i in range(n)])


@pytest.mark.parametrize("kind", TYPES)
def test_compact_moves_held_pages_down(kind):
    cache = Cache(kind, 3, 40, 2, 40, [300, 64, 0, 5, 130, 129, 0], 6, 35)
    _update(cache, release=[0], forks=[(4, 6), (5, 2)])
    for _ in range(2):
        book = cache.book()
        live = book.compact()
        cache.native.compact(cache.result.data_ptr(), **cache.kw())
        assert cache.result.tolist()[0] == live
        cache.same(book)


@pytest.mark.parametrize("pages,lengths", [(5, [0, 0]), (4, [256, 0]), (3000, [64 * 40 + i for i in range(20)])])
def test_compact_of_empty_full_and_large_pools(pages, lengths):
    cache = Cache("bf16", 2, pages, 1, 8, lengths, 45, 36)
    book = cache.book()
    live = book.compact()
    cache.native.compact(cache.result.data_ptr(), **cache.kw())
    assert cache.result.tolist()[0] == live
    cache.same(book)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("picked", [False, True])
def test_write_puts_rows_at_the_last_positions(kind, picked):
    lengths, counts = [100, 64, 3, 0, 130], [70, 64, 5, 0, 1]
    cache = Cache(kind, 3, 12, 2, 24, lengths, 4, 37)
    offsets = _offsets(counts)
    rows = offsets[-1]
    g = torch.Generator("cuda").manual_seed(38)
    kv = _normal(g, rows + 9, 2 * 48, dtype=cache.dtype)
    k, v = kv.split(48, 1)
    index = [(i * 7) % (rows + 9) for i in range(rows)]
    index[3], index[4] = -1, rows + 9
    book = cache.book()
    book.write(1, k, v, offsets, index if picked else None)
    at, which = _ints(offsets), _ints(index)
    cache.native.write(1, k.data_ptr(), v.data_ptr(), at.data_ptr(), rows, source_rows=len(kv),
                       index=which.data_ptr() if picked else 0, k_stride=kv.stride(0), v_stride=kv.stride(0), stream=_stream())
    cache.same(book)


def test_layers_further_apart_than_their_pages():
    """layer_stride: the layers' pools are slices of a larger buffer."""
    cache = Cache("f32", 2, 8, 1, 16, [70, 0], 3, 39)
    wide = torch.randn(2, 2, 8, PAGE, 16, device="cuda")  # [layer][keys, values]
    cache.keys, cache.values = wide[:, 0], wide[:, 1]
    cache.native.struct.keys, cache.native.struct.values = cache.keys.data_ptr(), cache.values.data_ptr()
    cache.native.struct.layer_stride = wide.stride(0)
    book = cache.book()
    assert book.update(forks=[(0, 1)], grow=[3, 3]) == [5, 0, 0]
    forks, grow = _ints([0, 1]), _ints([3, 3])
    cache.native.update(cache.result.data_ptr(), forks=forks.data_ptr(), fork_count=1, grow=grow.data_ptr(), **cache.kw())
    assert cache.result.tolist() == [5, 0, 0]
    assert torch.equal(cache.keys, book.keys) and torch.equal(cache.values, book.values)


# ---- together ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", TYPES)
def test_a_serving_run_of_all_of_them(kind):
    """Prompts enter packed, a beam forks, drafted trees are read and their accepted rows written, sequences leave, the pool is
    compacted: at each step the tree attention equals attention over the tokens kept on the side."""
    code, dtype = ref.TYPES[kind]
    h, kv, d, layers = 8, 2, 64, 2
    lengths = [90, 30, 64]
    cache = Cache(kind, layers, 24, kv, d, [0] * 5, 5, 41)
    g = torch.Generator("cuda").manual_seed(42)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    out = torch.empty(q.shape, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    ref.close(out, expected, size, q, k, d ** -0.5, 90)
    _update(cache, grow=lengths + [0, 0])
    offsets = _ints(_offsets(lengths + [0, 0]))
    cache.native.write(1, k.data_ptr(), v.data_ptr(), offsets.data_ptr(), len(q), k_stride=stride, v_stride=stride,
                       stream=_stream())
    at = _offsets(lengths)
    kept = [(k[a:b].clone(), v[a:b].clone()) for a, b in zip(at, at[1:])] + [None, None]
    _update(cache, forks=[(0, 3), (1, 4)])
    kept[3], kept[4] = kept[0], kept[1]
    for step in range(4):
        live = [s for s in range(5) if kept[s] is not None]
        nodes = [5 + s if s in live else 0 for s in range(5)]
        parents = [_branching(n, 50 + step * 5 + s) for s, n in enumerate(nodes)]
        (q, k, v), stride = _fused(g, sum(nodes), h, kv, d, dtype)
        out = torch.empty(q.shape, dtype=dtype, device="cuda")
        plan = native.TreeAttention(code, h, kv, d)
        room = _room(plan.workspace_bytes(5, len(q), 9, 200))
        starts, up = _offsets(nodes), _ints([p for row in parents for p in row])
        offsets = _ints(starts)
        plan.run(cache.native, 1, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(),
                 len(q), 9, 200, q_stride=stride, k_stride=stride, v_stride=stride, workspace=room.data_ptr(),
                 workspace_bytes=room.numel(), stream=_stream())
        chosen = []
        for s in live:
            rows = slice(starts[s], starts[s + 1])
            n, length = nodes[s], len(kept[s][0])
            keys, values = (torch.cat([kept[s][i], x[rows]]) for i, x in enumerate((k, v)))
            seen = torch.zeros(n, length + n, dtype=torch.bool, device="cuda")
            seen[:, :length] = True
            for i in range(n):
                seen[i, [length + j for j in ref.path(parents[s], i)]] = True
            expected, size = ref.attend(q[rows], keys, values, seen, d ** -0.5)
            ref.close(out[rows], expected, size, q[rows], keys, d ** -0.5, length + n)
            accepted = sorted(ref.path(parents[s], n - 1))
            chosen.append((s, [starts[s] + i for i in accepted]))
        grow = [0] * 5
        for s, rows in chosen:
            grow[s] = len(rows)
            kept[s] = tuple(torch.cat([x, y[rows]]) for x, y in zip(kept[s], (k, v)))
        _update(cache, grow=grow)
        offsets, index = _ints(_offsets(grow)), _ints([r for _, rows in chosen for r in rows])
        cache.native.write(1, k.data_ptr(), v.data_ptr(), offsets.data_ptr(), index.numel(), source_rows=len(q),
                           index=index.data_ptr(), k_stride=stride, v_stride=stride, stream=_stream())
        if step == 1:
            _update(cache, release=[0, 2])
            kept[0] = kept[2] = None
            book = cache.book()
            live_pages = book.compact()
            cache.native.compact(cache.result.data_ptr(), **cache.kw())
            assert cache.result.tolist()[0] == live_pages
            cache.same(book)


@pytest.mark.parametrize("kind", TYPES)
def test_captured_calls_replay_on_new_inputs(kind):
    """Each call captured into a graph on a side stream; the replay reads what the buffers hold then."""
    code, dtype = ref.TYPES[kind]
    h, kv, d, lengths = 8, 2, 64, [100, 29]
    cache = Cache(kind, 1, 12, kv, d, [0, 0], 5, 43)
    g = torch.Generator("cuda").manual_seed(44)
    (q, k, v), stride = _fused(g, 129, h, kv, d, dtype)
    out, tree_out = torch.empty(q.shape, dtype=dtype, device="cuda"), torch.empty(2, h, d, dtype=dtype, device="cuda")
    plan, step = native.PackedAttention(code, h, kv, d), native.TreeAttention(code, h, kv, d)
    room = _room(plan.workspace_bytes(2, 129) + step.workspace_bytes(2, 2, 1, 200))
    offsets, two, up, grow = _ints([0, 100, 129]), _ints([0, 1, 2]), _ints([-1, -1]), _ints(lengths)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        s = _stream()
        at = {"workspace": room.data_ptr(), "workspace_bytes": room.numel(), "stream": s}
        plan.run(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), 2, 129, q_stride=stride,
                 k_stride=stride, v_stride=stride, **at)
        cache.native.update(cache.result.data_ptr(), grow=grow.data_ptr(), **cache.kw())
        cache.native.write(0, k.data_ptr(), v.data_ptr(), offsets.data_ptr(), 129, k_stride=stride, v_stride=stride, stream=s)
        step.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), tree_out.data_ptr(), two.data_ptr(), up.data_ptr(),
                 2, 1, 200, q_stride=stride, k_stride=stride, v_stride=stride, **at)
        cache.native.compact(cache.result.data_ptr(), **cache.kw())
    for seed in (1, 2):
        fresh = _normal(torch.Generator("cuda").manual_seed(seed), 129, stride, dtype=dtype)
        q._base.copy_(fresh) if q._base is not None else None
        cache.table.fill_(-1), cache.lengths.zero_(), cache.refs.zero_()
        graph.replay()
        torch.cuda.synchronize()
        expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
        ref.close(out, expected, size, q, k, d ** -0.5, 100)
        expected, size = ref.tree(q[:2], k[:2], v[:2], [1, 1], [[-1], [-1]], cache.keys[0].view(cache.shape),
                                  cache.values[0].view(cache.shape), cache.table.tolist(), lengths, d ** -0.5)
        ref.close(tree_out, expected, size, q[:2], k, d ** -0.5, 200)
        assert cache.lengths.tolist() == lengths


def test_two_calls_side_by_side():
    """The same operators on two streams at once, each with its own workspace."""
    h, kv, d, lengths = 8, 1, 256, [200, 333]
    runs = []
    for i in range(2):
        g = torch.Generator("cuda").manual_seed(60 + i)
        (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, torch.float32)
        runs.append((q, k, v, stride, torch.empty(q.shape, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    kept = [_run_packed(native.F32, q, k, v, out, lengths, stride, stream=s.cuda_stream)
            for q, k, v, stride, out, s in runs for _ in range(3)]
    torch.cuda.synchronize()
    assert len(kept) == 6
    for q, k, v, _, out, _ in runs:
        expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
        ref.close(out, expected, size, q, k, d ** -0.5, 333)


@pytest.mark.parametrize("kind", TYPES)
def test_thousands_of_sequences(kind):
    """More sequences than a warp keeps in registers, many of them empty: prompts and decode steps."""
    code, dtype = ref.TYPES[kind]
    h, kv, d, n = 4, 2, 64, 3000
    lengths = [0 if i % 3 == 1 else (i * 7) % 20 if i % 50 else 90 + i % 60 for i in range(n)]
    g = torch.Generator("cuda").manual_seed(80)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    begin = 0
    for i, length in enumerate(lengths):
        if length and i % 97 in (0, 50):
            rows = slice(begin, begin + length)
            expected, size = ref.packed(q[rows], k[rows], v[rows], [length], d ** -0.5)
            ref.close(out[rows], expected, size, q[rows], k[rows], d ** -0.5, length)
        begin += length
    assert not bool(torch.isnan(out).any())
    cached = [(i * 11) % 150 for i in range(n)]
    cache = Cache(kind, 1, sum(-(-x // PAGE) for x in cached) + 2, kv, d, cached, 3, 81)
    nodes = [1 if i % 4 else 0 for i in range(n)]
    (q, k, v), stride = _fused(g, sum(nodes), h, kv, d, dtype)
    out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda")
    plan, offsets, up = native.TreeAttention(code, h, kv, d), _ints(_offsets(nodes)), _ints([-1] * sum(nodes))
    room = _room(plan.workspace_bytes(n, len(q), 1, 150))
    plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(),
             len(q), 1, 150, q_stride=stride, k_stride=stride, v_stride=stride, workspace=room.data_ptr(),
             workspace_bytes=room.numel(), stream=_stream())
    assert not bool(torch.isnan(out).any())
    at, table = _offsets(nodes), cache.table.tolist()
    for s in range(0, n, 61):
        rows = slice(at[s], at[s + 1])
        if nodes[s]:
            expected, size = ref.tree(q[rows], k[rows], v[rows], [1], [[-1]], cache.keys[0].view(cache.shape),
                                      cache.values[0].view(cache.shape), [table[s]], [cached[s]], d ** -0.5)
            ref.close(out[rows], expected, size, q[rows], cache.keys[0].view(-1, kv, d), d ** -0.5, 151)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(128, 1, 64), (70, 1, 128), (130, 2, 40)], ids=str)
def test_many_heads_over_one(kind, heads):
    """65 to 128 query heads over a kv head: a query tile is a single token."""
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    lengths = [67, 2]
    g = torch.Generator("cuda").manual_seed(70)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    ref.close(out, expected, size, q, k, d ** -0.5, 67)
    cache = Cache(kind, 1, 8, kv, d, [130, 0], 4, 71)
    _tree(cache, 0, h, kv, d, [3, 2], [[-1, 0, 0], [-1, -1]], 72, 130)


@pytest.mark.parametrize("kind", TYPES)
def test_caches_past_32_bits(kind):
    """Pages whose first element lies past 2^32 bytes and 2^31 elements of the pool, in every operator that takes pages."""
    code, dtype = ref.TYPES[kind]
    kv, d = 4, 128
    pages = 2 ** 31 // (PAGE * kv * d) + 40  # past 2^31 elements
    pools = [torch.empty(pages, PAGE, kv * d, dtype=dtype, device="cuda") for _ in range(2)]
    low, high = [0, 3], list(range(pages - 8, pages))
    g = torch.Generator("cuda").manual_seed(73)
    for pool in pools:
        for p in low + high:
            pool[p] = _normal(g, PAGE, kv * d, dtype=dtype)
    table, lengths = [[high[1], low[0], high[5], -1], [high[0], -1, -1, -1]], [150, 64]
    refs = [0] * pages
    for p in (high[1], low[0], high[5], high[0]):
        refs[p] = 1
    cache = Cache.__new__(Cache)
    cache.keys, cache.values = (pool[None] for pool in pools)
    cache.shape, cache.kind, cache.code, cache.dtype = (pages, PAGE, kv, d), kind, code, dtype
    cache.table, cache.lengths, cache.refs = _ints(table), _ints(lengths), _ints(refs)
    cache.native = native.PageCache(code, 1, pages, kv * d, 2, 4, pools[0].data_ptr(), pools[1].data_ptr(),
                                    cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr())
    cache.room, cache.result = _room(cache.native.workspace_bytes), _ints([0, 0, 0])
    _tree(cache, 0, 8, kv, d, [4, 1], [[-1, 0, 0, 1], [-1]], 74, 150)
    rows, offsets, index = _normal(g, 70, 2 * kv * d, dtype=dtype), _ints([0, 30, 33]), _ints([i * 2 for i in range(33)])
    k, v = rows.split(kv * d, 1)
    cache.native.write(0, k.data_ptr(), v.data_ptr(), offsets.data_ptr(), 33, source_rows=70, index=index.data_ptr(),
                       k_stride=rows.stride(0), v_stride=rows.stride(0), stream=_stream())
    for pool, source in ((pools[0], k), (pools[1], v)):
        for s, begin, count in ((0, 0, 30), (1, 30, 3)):
            for i in range(count):
                j = lengths[s] - count + i
                assert torch.equal(pool[table[s][j // PAGE], j % PAGE], source[(begin + i) * 2])
    kept = [[pool[p].clone() for p in (high[0], high[1], high[5])] for pool in pools]
    cache.native.compact(cache.result.data_ptr(), **cache.kw())
    assert cache.result.tolist()[0] == 4
    assert cache.table.tolist() == [[2, 0, 3, -1], [1, -1, -1, -1]] and cache.refs[:5].tolist() == [1, 1, 1, 1, 0]
    for pool, was in zip(pools, kept):
        for target, rows_of in zip((1, 2, 3), was):
            assert torch.equal(pool[target], rows_of)


def test_the_default_stream_and_no_stream_argument():
    g = torch.Generator("cuda").manual_seed(75)
    (q, k, v), stride = _fused(g, 90, 8, 1, 256, torch.float32)
    out = torch.empty(q.shape, device="cuda")
    torch.cuda.synchronize()
    kept = _run_packed(native.F32, q, k, v, out, [90], stride, stream=0)
    torch.cuda.synchronize()
    assert kept
    expected, size = ref.packed(q, k, v, [90], 1 / 16)
    ref.close(out, expected, size, q, k, 1 / 16, 90)


@pytest.mark.parametrize("kind", TYPES)
def test_long_prompts_and_caches(kind):
    """More tiles than any buffer holds, more units than CTAs: a few rows each against the formula."""
    code, dtype = ref.TYPES[kind]
    h, kv, d, n = 4, 2, 64, 6000
    g = torch.Generator("cuda").manual_seed(76)
    (q, k, v), stride = _fused(g, n + 7, h, kv, d, dtype)
    out = torch.empty(q.shape, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, [n, 7], stride)
    at = torch.tensor([0, 1, 63, 64, 2999, 4096, n - 1], device="cuda")
    seen = torch.arange(n, device="cuda") <= at[:, None]
    expected, size = ref.attend(q[at], k[:n], v[:n], seen, d ** -0.5)
    ref.close(out[at], expected, size, q[at], k, d ** -0.5, n)
    lengths = [9000, 17, 4500]
    cache = Cache(kind, 1, 220, kv, d, lengths, 145, 77)
    _tree(cache, 0, h, kv, d, [2, 5, 64], [_branching(i, i) for i in (2, 5, 64)], 78, 9000)


def test_host_memory_is_refused():
    q = torch.zeros(64, 8, 64)
    on = torch.zeros(64, 8, 64, device="cuda")
    plan, offsets = native.PackedAttention(native.F32, 8, 8, 64), _ints([0, 64])
    for args in ((q, on, on, on), (on, q, on, on), (on, on, on, q)):
        with pytest.raises(native.HFError) as e:
            plan.run(*(x.data_ptr() for x in args), offsets.data_ptr(), 1, 64, stream=_stream())
        assert e.value.code == native.HF_E_INVALID


# ---- keys that are not finite --------------------------------------------------------------------------------------


def _run_tree(cache, q, k, v, nodes, parents, max_length, layer=0):
    """The operator's rows and the formula's (with the rows' sizes)."""
    h, d = q.shape[1:]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    plan = native.TreeAttention(cache.code, h, k.shape[1], d)
    offsets, up = _ints(_offsets(nodes)), _ints([p for row in parents for p in row])
    room = _room(plan.workspace_bytes(len(nodes), len(q), max(nodes), max_length))
    plan.run(cache.native, layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(),
             len(q), max(nodes), max_length, workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.tree(q, k, v, nodes, parents, cache.keys[layer].view(cache.shape), cache.values[layer].view(cache.shape),
                              cache.table.tolist(), cache.lengths.tolist(), d ** -0.5)
    return out, expected, size


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 256), (4, 2, 64)], ids=str)
def test_a_key_alone_that_is_not_finite_in_a_prompt(kind, value, heads):
    """At every place of 16 in a tile, its value finite: what the rows in its own tile and in later ones come to is the
    formula's (a score of infinity or NaN makes the row NaN, one of minus infinity weighs nothing)."""
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    lengths = [200, 30]
    for place in range(16):
        g = torch.Generator("cuda").manual_seed(90 + place)
        (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
        k[64 + place + 16 * (place % 4), 0, 5] = value
        out = torch.full(q.shape, math.inf, dtype=dtype, device="cuda")
        _run_packed(code, q, k, v, out, lengths, stride)
        expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
        assert bool(torch.isnan(expected).any()) and bool(torch.isfinite(expected[:64]).all())
        ref.close(out, expected, size, q, k, d ** -0.5, max(lengths))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,nodes", [((8, 2, 128), 1), ((8, 1, 256), 5), ((4, 2, 64), 20)], ids=str)
def test_a_key_alone_that_is_not_finite_in_the_cache(kind, value, heads, nodes):
    """The same in a full cached page, for decode steps and trees whose keys lie with one CTA and with several."""
    h, kv, d = heads
    lengths = [300, 70, 4000]
    parents = [_branching(nodes, s) for s in range(3)]
    cache = Cache(kind, 1, 75, kv, d, lengths, 63, 91)
    g = torch.Generator("cuda").manual_seed(92)
    for place in range(16):
        q, k, v = (_normal(g, 3 * nodes, n, d, dtype=cache.dtype) for n in (h, kv, kv))
        at = []
        for s, j in ((0, 64 + place), (1, place + 48), (2, 640 + place)):
            page = cache.table.tolist()[s][j // PAGE]
            at.append((page, j % PAGE, cache.keys[0, page, j % PAGE, 3].item()))
            cache.keys[0, page, j % PAGE, 3] = value
        out, expected, size = _run_tree(cache, q, k, v, [nodes] * 3, parents, 4000)
        assert bool(torch.isnan(expected).any()) and (kv == 1 or bool(torch.isfinite(expected[:, h // kv:]).all()))
        everything = torch.cat([k, cache.keys[0].view(-1, kv, d)])
        ref.close(out, expected, size, q, everything, d ** -0.5, 4064)
        for page, j, was in at:
            cache.keys[0, page, j, 3] = was


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths", [[200, 1], [40, 1, 2], [700]], ids=str)
def test_prompt_rows_whose_every_score_is_minus_infinity(kind, lengths):
    """The formula has no weights for them: NaN, not the 0 of a row that attends to nothing. Later rows are finite."""
    code, dtype = ref.TYPES[kind]
    h, kv, d = 4, 2, 64
    g = torch.Generator("cuda").manual_seed(93)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    q[:, :, 5] = q[:, :, 5].abs() + 0.25
    for begin in _offsets(lengths)[:-1]:
        k[begin:begin + 3, 0, 5] = -math.inf
    out = torch.zeros(q.shape, dtype=dtype, device="cuda")
    _run_packed(code, q, k, v, out, lengths, stride)
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    assert bool(torch.isnan(expected[0, :2]).all()) and bool(torch.isfinite(expected[3:lengths[0]]).all())
    ref.close(out, expected, size, q, k, d ** -0.5, max(lengths))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("length", [20, 60, 300, 4000])
@pytest.mark.parametrize("nodes", [1, 7])
@pytest.mark.parametrize("lowest", [0.5, 1.0])
def test_tree_rows_whose_scores_are_minus_infinity(kind, length, nodes, lowest):
    """Half of the cache, or all of it and the nodes: the parts of a row in which every score is minus infinity weigh
    nothing beside others, and of nothing else the row is NaN."""
    h, kv, d = 4, 2, 64
    cache = Cache(kind, 1, 70, kv, d, [length, 33], 63, 94)
    g = torch.Generator("cuda").manual_seed(95)
    parents = [_branching(nodes, 3), _branching(nodes, 4)]
    q, k, v = (_normal(g, 2 * nodes, n, d, dtype=cache.dtype) for n in (h, kv, kv))
    q[:, :, 5] = q[:, :, 5].abs() + 0.25
    row = cache.table.tolist()[0]
    for j in range(int(length * lowest)):
        cache.keys[0, row[j // PAGE], j % PAGE, 5] = -math.inf
    if lowest == 1:
        k[:nodes, 0, 5] = -math.inf
    out, expected, size = _run_tree(cache, q, k, v, [nodes] * 2, parents, max(length, 33))
    assert bool(torch.isnan(expected[:nodes, :2]).all()) == (lowest == 1) and bool(torch.isfinite(expected[:, 2:]).all())
    everything = torch.cat([k, cache.keys[0].view(-1, kv, d)])
    ref.close(out, expected, size, q, everything, d ** -0.5, length + 64)


# ---- who calls -----------------------------------------------------------------------------------------------------


def test_a_thread_that_has_not_used_the_device():
    """A fresh thread has no current context of its own yet."""
    g = torch.Generator("cuda").manual_seed(96)
    (q, k, v), stride = _fused(g, 300, 8, 1, 256, torch.float32)
    out = torch.empty(q.shape, device="cuda")
    stream, failed = _stream(), []
    plan, offsets = native.PackedAttention(native.F32, 8, 1, 256), _ints([0, 300])
    room = _room(plan.workspace_bytes(1, 300))
    torch.cuda.synchronize()

    def call():
        try:
            plan.run(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), 1, 300, q_stride=stride,
                     k_stride=stride, v_stride=stride, workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=stream)
        except native.HFError as e:
            failed.append(e)

    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not failed
    expected, size = ref.packed(q, k, v, [300], 1 / 16)
    ref.close(out, expected, size, q, k, 1 / 16, 300)


@pytest.mark.parametrize("kind,n", [("bf16", 120064), ("f16", 20096), ("f32", 40064)])
def test_rows_taken_again_over_many_keys(kind, n):
    """An infinite value near a long prompt's end: the rows of its tile are taken again over all of their keys, a warp's 32
    (fp32: 16) in 0.3 to 1.7 s, and what waits for them waits on. (bf16: by the second of a CTA's two query tiles.)"""
    code, dtype = ref.TYPES[kind]
    g = torch.Generator("cuda").manual_seed(99)
    q, k, v = (_normal(g, n, 1, 8, dtype=dtype) for _ in range(3))
    bad = n - 30
    v[bad, 0, 3] = math.inf
    out = torch.empty_like(q)
    kept = _run_packed(code, q, k, v, out, [n], 8)
    torch.cuda.synchronize()
    assert kept
    at = torch.tensor([0, n // 2, n - 128, n - 65, bad - 1, bad, n - 1], device="cuda")
    seen = torch.arange(n, device="cuda") <= at[:, None]
    expected, size = ref.attend(q[at], k, v, seen, 8 ** -0.5)
    fine = torch.isfinite(expected)
    assert int((~fine).sum()) == 2 and torch.equal(torch.isfinite(out[at]), fine)
    tol = ref.tolerance(expected.nan_to_num(0, 0, 0), size.nan_to_num(0, 0, 0), q, k, 8 ** -0.5, n, dtype)
    assert bool(((out[at].double() - expected).abs() <= tol)[fine].all())
    assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("kind", TYPES)
def test_a_call_repeated_gives_the_same_bits(kind):
    code, dtype = ref.TYPES[kind]
    h, kv, d, lengths = 8, 2, 128, [900, 3, 0, 400, 131]
    g = torch.Generator("cuda").manual_seed(97)
    (q, k, v), stride = _fused(g, sum(lengths), h, kv, d, dtype)
    prompts = [torch.empty(q.shape, dtype=dtype, device="cuda") for _ in range(4)]
    for out in prompts:
        _run_packed(code, q, k, v, out, lengths, stride)
    cached = [3000, 700, 0, 64, 1900]
    cache = Cache(kind, 1, 100, kv, d, cached, 47, 98)
    trees = []
    for nodes in (1, 12):
        q, k, v = (_normal(g, 5 * nodes, n, d, dtype=dtype) for n in (h, kv, kv))
        trees.append([_run_tree(cache, q, k, v, [nodes] * 5, [_branching(nodes, s) for s in range(5)], 3000)[0]
                      for _ in range(4)])
    for first, *others in (prompts, *trees):
        for other in others:
            assert torch.equal(first.view(torch.uint8), other.view(torch.uint8))

# ---- what the documentation allows ---------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("sequences", [1, 5, 200])
def test_a_batch_without_a_row(kind, sequences):
    """Every sequence is empty: nothing is read or written, in calls of many rows and of few."""
    code, dtype = ref.TYPES[kind]
    for rows in (4, 900):
        q, k, v = (torch.full((rows, n, 64), math.nan, dtype=dtype, device="cuda") for n in (8, 2, 2))
        out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
        _run_packed(code, q, k, v, out, [0] * sequences, 0, begin=rows // 2)
        assert bool((out == 7.0).all())
        cache = Cache(kind, 1, 3, 2, 64, [0] * sequences, 2, 101)
        plan, offsets, up = native.TreeAttention(code, 8, 2, 64), _ints([rows // 2] * (sequences + 1)), _ints([-1] * rows)
        room = _room(plan.workspace_bytes(sequences, rows, 5, 128))
        plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(), up.data_ptr(),
                 rows, 5, 128, workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=_stream())
        assert bool((out == 7.0).all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads", [(8, 1, 256), (4, 2, 40), (16, 4, 128)], ids=str)
@pytest.mark.parametrize("lengths", [[20, 5], [300, 1, 77], [700] * 6], ids=str)
def test_rows_of_every_operand_further_apart(kind, heads, lengths):
    """A row stride of its own for q, k, v and out; what lies between out's rows stays."""
    code, dtype = ref.TYPES[kind]
    h, kv, d = heads
    rows = sum(lengths)
    g = torch.Generator("cuda").manual_seed(102)
    wide = [_normal(g, rows, n * d + 8 * (i + 1), dtype=dtype) for i, n in enumerate((h, kv, kv, h))]
    wide[3].fill_(7.0)
    q, k, v, out = (x[:, 8 * (i + 1):].unflatten(1, (-1, d)) for i, x in enumerate(wide))
    offsets = _ints(_offsets(lengths))
    strides = dict(zip(("q_stride", "k_stride", "v_stride", "out_stride"), (x.stride(0) for x in wide)))
    plan = native.PackedAttention(code, h, kv, d)
    room = _room(plan.workspace_bytes(len(lengths), rows))
    plan.run(*(x.data_ptr() for x in (q, k, v, out)), offsets.data_ptr(), len(lengths), rows, **strides,
             workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.packed(q, k, v, lengths, d ** -0.5)
    ref.close(out, expected, size, q, k, d ** -0.5, max(lengths))
    assert bool((wide[3][:, :32] == 7.0).all())
    nodes = [min(n, 9) for n in lengths]
    cache = Cache(kind, 1, 40, kv, d, [200, 70, 0, 333, 64, 1][:len(lengths)], 6, 103)
    parents = [_branching(n, i) for i, n in enumerate(nodes)]
    wide[3].fill_(7.0)
    used, step = sum(nodes), native.TreeAttention(code, h, kv, d)
    offsets, up = _ints(_offsets(nodes)), _ints([p for row in parents for p in row])
    room = _room(step.workspace_bytes(len(nodes), used, 9, 333))
    step.run(cache.native, 0, *(x.data_ptr() for x in (q, k, v, out)), offsets.data_ptr(), up.data_ptr(), used, 9, 333, **strides,
             workspace=room.data_ptr(), workspace_bytes=room.numel(), stream=_stream())
    expected, size = ref.tree(q[:used], k[:used], v[:used], nodes, parents, cache.keys[0].view(cache.shape),
                              cache.values[0].view(cache.shape), cache.table.tolist(), cache.lengths.tolist(), d ** -0.5)
    everything = torch.cat([k[:used], cache.keys[0].view(-1, kv, d)])
    ref.close(out[:used], expected, size, q[:used], everything, d ** -0.5, 342)
    assert bool((wide[3][:, :32] == 7.0).all()) and bool((wide[3][used:] == 7.0).all())


@pytest.mark.parametrize("kind", TYPES)
def test_graphs_side_by_side(kind):
    """Two captured steps replayed at once on two streams, a workspace each, over one cache."""
    code, dtype = ref.TYPES[kind]
    h, kv, d, lengths = 8, 2, 128, [1500, 300, 64]
    cache = Cache(kind, 1, 40, kv, d, lengths, 24, 104)
    g = torch.Generator("cuda").manual_seed(105)
    runs = []
    for nodes in (1, 6):
        q, k, v = (_normal(g, 3 * nodes, n, d, dtype=dtype) for n in (h, kv, kv))
        out, parents = torch.empty_like(q), [_branching(nodes, s) for s in range(3)]
        plan = native.TreeAttention(code, h, kv, d)
        offsets, up = _ints(_offsets([nodes] * 3)), _ints([p for row in parents for p in row])
        room = _room(plan.workspace_bytes(3, len(q), nodes, 1500))
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(20):
                plan.run(cache.native, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), offsets.data_ptr(),
                         up.data_ptr(), len(q), nodes, 1500, workspace=room.data_ptr(), workspace_bytes=room.numel(),
                         stream=_stream())
        runs.append((graph, stream, q, k, v, out, nodes, parents, plan, offsets, up, room))
    for _ in range(5):
        for graph, stream, *_rest in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, q, k, v, out, nodes, parents, *_rest in runs:
        expected, size = ref.tree(q, k, v, [nodes] * 3, parents, cache.keys[0].view(cache.shape),
                                  cache.values[0].view(cache.shape), cache.table.tolist(), lengths, d ** -0.5)
        ref.close(out, expected, size, q, torch.cat([k, cache.keys[0].view(-1, kv, d)]), d ** -0.5, 1506)


@pytest.mark.parametrize("scale", [1e-3, 1e-6, 1e-9])
def test_fp32_channels_far_below_the_others(scale):
    """Every 17th channel of the values is `scale` times as large as the others. Two fp16 halves under their tile's exponent are
    off by half of 2^-24 where the largest value is at least 2^14 (trees: 2^10 of their sample's), so the error is the
    tolerance of the channel itself and 2^-39 (2^-35) of the largest value: weights sum to one."""
    h, d = 8, 256
    g = torch.Generator("cuda").manual_seed(106)
    (q, k, v), stride = _fused(g, 340, h, 1, d, torch.float32)
    v[:, :, 3::17] *= scale
    out = torch.empty(q.shape, device="cuda")
    _run_packed(native.F32, q, k, v, out, [300, 40], stride)
    expected, size = ref.packed(q, k, v, [300, 40], 1 / 16)
    tol = ref.tolerance(expected, size, q, k, 1 / 16, 300, torch.float32) + 2.0 ** -39 * float(v.abs().max())
    assert bool(((out.double() - expected).abs() <= tol).all())
    cache = Cache("f32", 1, 24, 1, d, [1000, 300], 20, 107)
    cache.values[:, :, :, 3::17] *= scale
    q, k, v = (_normal(g, 20, n, d, dtype=torch.float32) for n in (h, 1, 1))
    v[:, :, 3::17] *= scale
    out, expected, size = _run_tree(cache, q, k, v, [10, 10], [_branching(10, 1), _branching(10, 2)], 1000)
    everything = torch.cat([k, cache.keys[0].view(-1, 1, d)])
    tol = ref.tolerance(expected, size, q, everything, 1 / 16, 1010, torch.float32)
    tol += 2.0 ** -35 * float(cache.values.abs().max())
    assert bool(((out.double() - expected).abs() <= tol).all())
