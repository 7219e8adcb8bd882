"""A plan of the serving operators that two callers share (CPU only: the library is a stand-in that records its calls)."""
import pytest

from huggingfaceeacp_b200 import native

NAMES = ("q", "k", "v", "out", "offsets", "rows", "q_stride", "k_stride", "v_stride", "out_stride", "workspace",
         "workspace_bytes")


class Library:
    """Runs `between` inside a call, as another thread's call can while this one is in the library; then reads the call."""

    def __init__(self):
        self.between, self.calls = None, []

    def _call(self, struct, extra=()):
        between, self.between = self.between, None
        if between:
            between()
        self.calls.append({n: getattr(struct, n) for n in NAMES + tuple(extra)})
        return 0

    def hf_cuda_attention_packed(self, call, stream):
        return self._call(call._obj, ("sequences",))

    def hf_cuda_attention_tree(self, cache, call, stream):
        return self._call(call._obj, ("max_nodes", "max_length", "layer", "parents"))

    def hf_cuda_attention_packed_workspace(self, call, size):
        return 0

    def hf_cuda_attention_tree_workspace(self, cache, call, size):
        return 0


def _arguments(base, **more):
    return {**{n: base + 16 * i for i, n in enumerate(NAMES)}, **more}


@pytest.mark.parametrize("asks", [False, True], ids=["run", "workspace_bytes"])
def test_prompts(asks):
    plan = native.PackedAttention(native.F32, 8, 1, 256)
    plan.lib = Library()
    mine, theirs = _arguments(1 << 20, sequences=3), _arguments(1 << 30, sequences=9)
    plan.lib.between = (lambda: plan.workspace_bytes(77, 777)) if asks else (lambda: plan.run(**theirs))
    plan.run(**mine)
    assert plan.lib.calls == ([mine] if asks else [theirs, mine])


@pytest.mark.parametrize("asks", [False, True], ids=["run", "workspace_bytes"])
def test_trees(asks):
    plan = native.TreeAttention(native.F16, 8, 2, 64)
    plan.lib = Library()
    cache = native.PageCache(native.F16, 4, 8, 128, 3, 4, 0, 0, 0, 0, 0)
    mine = _arguments(1 << 20, max_nodes=5, max_length=200, layer=1, parents=1 << 22)
    theirs = _arguments(1 << 30, max_nodes=9, max_length=100, layer=2, parents=1 << 23)
    plan.lib.between = (lambda: plan.workspace_bytes(7, 777, 3, 33)) if asks else (lambda: plan.run(cache, **theirs))
    plan.run(cache, **mine)
    assert plan.lib.calls == ([mine] if asks else [theirs, mine])


def test_what_the_library_gets():
    """Every field of both calls, as the header lays them out."""
    plan = native.PackedAttention(native.BF16, 6, 3, 40, scale=0.5)
    seen = []
    plan.lib = type("L", (), {"hf_cuda_attention_packed": lambda self, call, stream: seen.append(call._obj) or 0})()
    plan.run(1, 2, 3, 4, 5, 6, 7, q_stride=8, k_stride=9, v_stride=10, out_stride=11, workspace=12, workspace_bytes=13)
    want = dict(dtype=native.BF16, heads=6, kv_heads=3, head_width=40, sequences=6, rows=7, scale=0.5, q=1, k=2, v=3, out=4,
                q_stride=8, k_stride=9, v_stride=10, out_stride=11, offsets=5, workspace=12, workspace_bytes=13)
    assert {n: getattr(seen[0], n) for n, _ in native.PackedStruct._fields_} == want
    step = native.TreeAttention(native.BF16, 6, 3, 40, scale=0.5)
    step.lib = type("L", (), {"hf_cuda_attention_tree": lambda self, cache, call, stream: seen.append(call._obj) or 0})()
    cache = native.PageCache(native.BF16, 4, 8, 120, 3, 4, 0, 0, 0, 0, 0)
    step.run(cache, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, q_stride=16, k_stride=17, v_stride=18, out_stride=19, workspace=20,
             workspace_bytes=21)
    want = dict(heads=6, kv_heads=3, head_width=40, rows=8, max_nodes=9, max_length=10, layer=1, scale=0.5, q=2, k=3, v=4,
                out=5, q_stride=16, k_stride=17, v_stride=18, out_stride=19, offsets=6, parents=7, workspace=20,
                workspace_bytes=21)
    assert {n: getattr(seen[1], n) for n, _ in native.TreeStruct._fields_} == want
