"""examples/distill_lm.py: the three language-model operators in a training
step, on the device against the plain CPU path, eager and as a CUDA graph."""
import pytest

import xdna_train
from examples import distill_lm

SMALL = dict(vocab=200, width=64, hidden=168, blocks=2, top=8, batch=8, length=12)


def test_student_learns_on_cpu():
    losses = distill_lm.train(steps=25, device="cpu", **SMALL)
    assert all(v == v for v in losses) and losses[-1] < 0.6 * losses[0]


@pytest.mark.gpu
def test_device_follows_the_cpu_path(cuda):
    ref = distill_lm.train(steps=25, device="cpu", **SMALL)
    xdna_train.reset_mapped_cpu_stats()
    got = distill_lm.train(steps=25, device="xdna", **SMALL)
    stats = xdna_train.kernel_stats()
    for k in ("lm.embedding", "lm.embedding_bwd", "lm.gated_mlp", "lm.gated_mlp_bwd", "lm.distill", "lm.distill_bwd"):
        assert stats.get(k, 0) > 0, (k, stats)
    # the same mathematics; the CPU path rounds more tensors to bf16 on the way, and training amplifies differences
    assert abs(got[0] - ref[0]) <= 0.01 * ref[0]
    assert all(abs(a - b) <= 0.06 * b for a, b in zip(got, ref)), list(zip(got, ref))
    assert xdna_train.device_status(0) == 0


@pytest.mark.gpu
def test_whole_step_as_a_graph(cuda):
    eager = distill_lm.train(steps=12, device="xdna", **SMALL)
    graphed = distill_lm.train(steps=12, device="xdna", graph=True, **SMALL)
    # the graph's warm-up takes one more step on the first batch
    assert graphed[-1] < 0.8 * eager[0] and all(v == v for v in graphed)
    assert abs(graphed[0] - eager[0]) <= 0.35 * eager[0]
