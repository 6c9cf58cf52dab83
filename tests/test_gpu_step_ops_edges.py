"""GPU: calls of the scheduler-step operators at the edges of what they allow:
queries that are not finite, against the rule that a row's values reach that
row alone, and the ends of int32 in the fog's boundary, against 64 bits."""

import pytest
import torch

from tests.test_gpu_step_ops import _Case, _i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield


@pytest.fixture(autouse=True)
def _no_status():
    from kessie_b200 import ops
    ops.read_device_status()
    yield
    assert ops.read_device_status() == 0, "device status bits left by a test that expects none"


# ------------------------------------------------------------------ queries that are not finite
# one sequence, whose tiles the whole grid cuts; and more tiles than a plan can cut (one boundary a CTA), single
# (3 tokens of 4 heads) and pair ones
BROKEN = {"cut": ([40], [6000]), "cut single": ([3], [6000]),
          "many": ([3, 70] * 150, [500 + 3 * i for i in range(300)])}


@pytest.mark.parametrize("fog", ["none", "values", "scores"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths", list(BROKEN))
def test_chunks_queries_that_are_not_finite_reach_their_rows_alone(lengths, dt, fog):
    """A NaN in a query makes all its scores NaN, an infinite one makes scores
    of both signs, whose softmax is inf - inf: the row is NaN, every other row
    is as it was, bit for bit."""
    from kessie_b200 import ops
    q_lens, kv_lens = BROKEN[lengths]
    c = _Case(71, q_lens, kv_lens, 8, 2, 64, 16, dt)
    kw = {"none": dict(), "values": dict(clear_start=_i32([n * 3 // 4 for n in kv_lens])),
          "scores": dict(bias=ops.FogBias(1.5, 0.5, dtype=torch.float32), fog_alpha=0.0)}[fog]
    want = c.run(**kw)
    broken = torch.zeros(c.q.shape[:2], dtype=torch.bool, device="cuda")
    for b, row in enumerate(c.start[:-1].tolist()):
        n = q_lens[b]
        c.q[row, b % 8, 5] = float("nan")
        c.q[row + n - 1, (b + 3) % 8] = float("inf")
        c.q[row + n // 2, (b + 6) % 8, b % 64] = float("-inf")
        broken[row, b % 8] = broken[row + n - 1, (b + 3) % 8] = broken[row + n // 2, (b + 6) % 8] = True
    got = c.run(**kw)
    assert got[broken].isnan().all(), f"{(~got[broken].isnan().all(-1)).sum().item()} of {broken.sum().item()} rows"
    assert torch.equal(got[~broken], want[~broken])


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_chunks_rows_without_keys_are_zero_whatever_their_queries(dt):
    c = _Case(72, [200, 3], [50, 0], 8, 2, 128, 16, dt)
    c.q[:150] = float("nan")
    c.q[200:] = float("inf")
    out = c.run(out=torch.full_like(c.q, 9.0))
    assert out[:150].count_nonzero() == 0 and out[200:].count_nonzero() == 0
    clean = _Case(72, [200, 3], [50, 0], 8, 2, 128, 16, dt)
    assert torch.equal(out[150:200], clean.run()[150:200])


# ------------------------------------------------------------------ the fog's boundary
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("clear", [2 ** 31 - 1, 2 ** 31 - 127, 2 ** 31 - 128, -2 ** 31, 1, 2])
def test_chunks_fog_boundary_anywhere_in_int32(clear, dt):
    """All keys fogged, far past the last of them, or none: single and pair
    tiles, cut ones among them (pieces from key 0 and from later keys)."""
    q_lens, kv_lens = [1, 70, 3, 200], [5000, 300, 40, 9000]
    c = _Case(73, q_lens, kv_lens, 8, 2, 64, 16, dt)
    c.check(c.run(clear_start=_i32([clear] * 4), fog_alpha=0.02), clear=[min(max(clear, 0), 2 ** 31 - 1)] * 4,
            alpha=0.02)
