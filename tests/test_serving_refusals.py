"""What the serving operators refuse on the host, before anything touches a GPU (CPU only: no call here gets as far as a
device pointer)."""
import pytest

from huggingfaceeacp_b200 import native

GOOD = 1 << 20  # an aligned address that no call here follows


def _cache(**changes):
    values = dict(dtype=native.BF16, layers=2, pages=8, kv_width=128, sequences=3, table_stride=4, keys=GOOD, values=GOOD,
                  table=GOOD, lengths=GOOD, refs=GOOD, layer_stride=0)
    values.update(changes)
    return native.PageCache(**values)


def _code(call, *args, **kw):
    with pytest.raises(native.HFError) as e:
        call(*args, **kw)
    return e.value.code


@pytest.mark.parametrize("changes,code", [
    ({"dtype": 3}, native.HF_E_INVALID), ({"dtype": -1}, native.HF_E_INVALID), ({"layers": 0}, native.HF_E_INVALID),
    ({"pages": 0}, native.HF_E_INVALID), ({"sequences": 0}, native.HF_E_INVALID), ({"table_stride": 0}, native.HF_E_INVALID),
    ({"table_stride": 1 << 21}, native.HF_E_INVALID), ({"kv_width": 4}, native.HF_E_SHAPE),
    ({"kv_width": 132}, native.HF_E_SHAPE), ({"layer_stride": 100}, native.HF_E_INVALID),
    ({"layer_stride": 8 * 64 * 128 + 4}, native.HF_E_INVALID),
], ids=str)
def test_cache_sizes(changes, code):
    cache = _cache(**changes)
    with pytest.raises(native.HFError) as e:
        cache.workspace_bytes
    assert e.value.code == code
    assert _code(cache.compact, GOOD, GOOD, 1 << 30) == code


@pytest.mark.parametrize("missing", ["keys", "values", "table", "lengths", "refs"])
def test_cache_pointers(missing):
    cache = _cache(**{missing: 0})
    assert _code(cache.update, GOOD, GOOD, 1 << 30) == native.HF_E_INVALID
    assert _code(cache.compact, GOOD, GOOD, 1 << 30) == native.HF_E_INVALID
    assert _code(cache.write, 0, GOOD, GOOD, GOOD, 5) == native.HF_E_INVALID
    if missing in ("keys", "values"):
        assert _code(_cache(**{missing: GOOD + 8}).compact, GOOD, GOOD, 1 << 30) == native.HF_E_INVALID


def test_page_steps():
    cache = _cache()
    size = cache.workspace_bytes
    assert size > 0
    assert _code(cache.update, GOOD, GOOD, size - 1) == native.HF_E_CAPACITY
    assert _code(cache.compact, GOOD, GOOD, size - 1) == native.HF_E_CAPACITY
    for bad in ({"result": 0}, {"workspace": 0}, {"workspace": GOOD + 4}, {"releases": -1}, {"releases": 4, "release": GOOD},
                {"releases": 1}, {"fork_count": 1}, {"fork_count": 4, "forks": GOOD}, {"fork_count": -2}):
        args = {"result": GOOD, "workspace": GOOD, "workspace_bytes": size, **bad}
        assert _code(cache.update, **args) == native.HF_E_INVALID
    for bad in ({"layer": 2}, {"layer": -1}, {"k": 0}, {"v": GOOD + 2}, {"offsets": 0}, {"rows": -1}, {"source_rows": -1},
                {"k_stride": 120}, {"v_stride": 132}):
        args = {"layer": 0, "k": GOOD, "v": GOOD, "offsets": GOOD, "rows": 5, **bad}
        assert _code(cache.write, **args) == native.HF_E_INVALID
    cache.write(0, GOOD, GOOD, GOOD, 0)  # no rows: nothing to do


@pytest.mark.parametrize("heads,code", [((6, 4, 64), native.HF_E_SHAPE), ((4, 4, 12), native.HF_E_SHAPE),
                                        ((4, 4, 264), native.HF_E_SHAPE), ((129, 1, 64), native.HF_E_SHAPE),
                                        ((0, 1, 64), native.HF_E_INVALID), ((4, 0, 64), native.HF_E_INVALID)], ids=str)
def test_attention_heads(heads, code):
    plan = native.PackedAttention(native.F16, *heads, scale=1.0)
    assert _code(plan.workspace_bytes, 2, 64) == code
    assert _code(plan.run, GOOD, GOOD, GOOD, GOOD, GOOD, 2, 64, workspace=GOOD, workspace_bytes=1 << 40) == code


@pytest.mark.parametrize("bad", [{"q": 0}, {"k": 0}, {"v": 0}, {"out": 0}, {"offsets": 0}, {"q": GOOD + 8}, {"out": GOOD + 2},
                                 {"sequences": 0}, {"rows": 0}, {"q_stride": 500}, {"k_stride": 132}, {"out_stride": -512}],
                         ids=str)
@pytest.mark.parametrize("kind", [native.F32, native.BF16, native.F16])
def test_packed_arguments(bad, kind):
    args = {"q": GOOD, "k": GOOD, "v": GOOD, "out": GOOD, "offsets": GOOD, "sequences": 2, "rows": 64, "workspace": GOOD,
            "workspace_bytes": 1 << 40, **bad}
    if kind == native.F32 and "k_stride" in bad:
        args["k_stride"] = 129  # four bytes off a 16-byte border
    assert _code(native.PackedAttention(kind, 8, 2, 64).run, **args) == native.HF_E_INVALID


def test_packed_scale_and_type():
    for scale in (float("nan"), float("inf"), 0.0, -0.5):
        assert _code(native.PackedAttention(native.F32, 8, 2, 64, scale=scale).workspace_bytes, 1, 1) == native.HF_E_INVALID
    assert _code(native.PackedAttention(5, 8, 2, 64).workspace_bytes, 1, 1) == native.HF_E_INVALID


@pytest.mark.parametrize("bad,code", [
    ({"q": 0}, native.HF_E_INVALID), ({"parents": 0}, native.HF_E_INVALID), ({"offsets": 0}, native.HF_E_INVALID),
    ({"v": GOOD + 4}, native.HF_E_INVALID), ({"rows": 0}, native.HF_E_INVALID), ({"max_nodes": 0}, native.HF_E_INVALID),
    ({"max_nodes": 65}, native.HF_E_SHAPE), ({"max_length": -1}, native.HF_E_INVALID), ({"layer": 2}, native.HF_E_INVALID),
    ({"layer": -1}, native.HF_E_INVALID), ({"q_stride": 8}, native.HF_E_INVALID),
], ids=str)
def test_tree_arguments(bad, code):
    args = {"cache": _cache(), "layer": 0, "q": GOOD, "k": GOOD, "v": GOOD, "out": GOOD, "offsets": GOOD, "parents": GOOD,
            "rows": 9, "max_nodes": 5, "max_length": 200, "workspace": GOOD, "workspace_bytes": 1 << 40, **bad}
    assert _code(native.TreeAttention(native.BF16, 8, 2, 64).run, **args) == code


def test_tree_cache_must_match():
    args = {"layer": 0, "q": GOOD, "k": GOOD, "v": GOOD, "out": GOOD, "offsets": GOOD, "parents": GOOD, "rows": 9,
            "max_nodes": 5, "max_length": 200, "workspace": GOOD, "workspace_bytes": 1 << 40}
    assert _code(native.TreeAttention(native.BF16, 8, 2, 64).run, cache=_cache(kv_width=64), **args) == native.HF_E_SHAPE
    assert _code(native.TreeAttention(native.F32, 8, 2, 64).run, cache=_cache(), **args) == native.HF_E_INVALID


def test_int32_arrays_off_their_border():
    """Refused ahead of the workspace's size: a kernel would fault on them."""
    for name in ("table", "lengths", "refs"):
        cache = _cache(**{name: GOOD + 2})
        assert _code(cache.update, GOOD, GOOD, 0) == native.HF_E_INVALID
        assert _code(cache.compact, GOOD, GOOD, 0) == native.HF_E_INVALID
        assert _code(cache.write, 0, GOOD, GOOD, GOOD, 5) == native.HF_E_INVALID
    lists = {"result": GOOD, "release": GOOD, "releases": 1, "forks": GOOD, "fork_count": 1, "grow": GOOD}
    assert _code(_cache().update, **lists, workspace=GOOD, workspace_bytes=0) == native.HF_E_CAPACITY
    for name in ("result", "release", "forks", "grow"):
        bad = {**lists, name: GOOD + 1}
        assert _code(_cache().update, **bad, workspace=GOOD, workspace_bytes=0) == native.HF_E_INVALID
    assert _code(_cache().compact, GOOD + 3, GOOD, 0) == native.HF_E_INVALID
    for name in ("offsets", "index"):
        args = {"layer": 0, "k": GOOD, "v": GOOD, "offsets": GOOD, "rows": 0, "index": GOOD, name: GOOD + 2}
        assert _code(_cache().write, **args) == native.HF_E_INVALID
    rows = {"q": GOOD, "k": GOOD, "v": GOOD, "out": GOOD, "offsets": GOOD, "rows": 9, "workspace": GOOD, "workspace_bytes": 0}
    prompt, step = native.PackedAttention(native.F32, 8, 2, 64), native.TreeAttention(native.BF16, 8, 2, 64)
    assert _code(prompt.run, **rows, sequences=2) == native.HF_E_CAPACITY
    assert _code(prompt.run, **{**rows, "offsets": GOOD + 2}, sequences=2) == native.HF_E_INVALID
    tree = {**rows, "cache": _cache(), "layer": 0, "parents": GOOD, "max_nodes": 5, "max_length": 200}
    assert _code(step.run, **tree) == native.HF_E_CAPACITY
    for bad in ({"offsets": GOOD + 1}, {"parents": GOOD + 2}, {"cache": _cache(table=GOOD + 1)},
                {"cache": _cache(lengths=GOOD + 2)}):
        assert _code(step.run, **{**tree, **bad}) == native.HF_E_INVALID
