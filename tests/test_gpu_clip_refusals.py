"""What gradient clipping refuses once there are tensors to look at."""
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
