"""What gradient clipping refuses once there are tensors to look at."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HYPER = (1e-3, 0.9, 0.999, 1e-8, 0.01, 1e-2, 31.6)


def tensors(rt, *sizes):
    return [rt.tensorFromData(np.full(n, 0.5, np.float32), [n], "float32")["id"] for n in sizes]


@pytest.mark.parametrize("step", ["adamWClipStepMulti", "adamClipStepMulti"])
@pytest.mark.parametrize("side", range(4), ids=["params", "grads", "exp_avgs", "exp_avg_sqs"])
def test_a_clipped_step_refuses_a_tensor_listed_twice(cuda_rt, step, side):
    """As clipping followed by the step does: a gradient listed twice would be
    scaled twice there, and a parameter or moment be updated by two CTAs at once."""
    rt = cuda_rt
    lists = [tensors(rt, 5, 5) for _ in range(4)]
    lists[side][1] = lists[side][0]
    before = [rt.toList(t) for t in sum(lists, [])]
    with pytest.raises(RuntimeError, match="twice"):
        getattr(rt, step)(*lists, *HYPER, 1.0)
    assert [rt.toList(t) for t in sum(lists, [])] == before


def test_a_clipped_step_refuses_one_tensor_in_two_lists(cuda_rt):
    rt = cuda_rt
    for a in range(4):
        for b in range(a):
            lists = [tensors(rt, 5, 70) for _ in range(4)]
            lists[a][1] = lists[b][1]
            with pytest.raises(RuntimeError, match="twice"):
                rt.adamWClipStepMulti(*lists, *HYPER, 1.0)
    lists = [tensors(rt, 5, 70) for _ in range(4)]
    assert rt.adamWClipStepMulti(*lists, *HYPER, 1.0)["shape"] == [2]


def test_tensor_lists_are_refused_in_a_capture(cuda_rt):
    """Their table is copied from host memory that is gone when a graph replays
    the copy; a group made before the capture is what a captured step uses."""
    rt = cuda_rt
    L = rt.lib
    lists = [tensors(rt, 40, 7) for _ in range(4)]
    p = ctypes.c_void_p()
    assert L.tp_alloc(64, ctypes.byref(p)) == 0
    rows, sizes, g = (ctypes.c_void_p * 1)(p.value), (ctypes.c_int64 * 1)(16), ctypes.c_int64()
    rt.synchronize()
    assert L.tp_graph_begin() == 0
    said = []
    for call in (lambda: rt.clipGradNormMulti(lists[0], 1.0), lambda: rt.adamWClipStepMulti(*lists, *HYPER, 1.0),
                 lambda: rt.adamClipStepMulti(*lists, *HYPER, 1.0), lambda: rt.adamWStepMulti(*lists, *HYPER)):
        try:
            call()
            said.append("accepted")
        except RuntimeError as e:
            said.append(str(e))
    status = L.tpk_group_create(1, rows, rows, rows, rows, sizes, ctypes.byref(g))
    said.append("accepted" if status == 0 else L.tp_last_error().decode())
    assert L.tp_memset(p.value, 0, 64) == 0
    graph = ctypes.c_int64()
    assert L.tp_graph_end(ctypes.byref(graph)) == 0, L.tp_last_error()
    assert all("capture" in s for s in said), said
    assert L.tp_graph_launch(graph.value) == 0
    rt.synchronize()
    assert L.tp_graph_destroy(graph.value) == 0 and L.tp_free(p.value) == 0
    assert all(rt.toList(t) == [0.5] * n for side in lists for t, n in zip(side, (40, 7)))
    assert rt.clipGradNormMulti(lists[1], 1.0)["shape"] == [2]  # and outside of it
