"""GPU: the decode's rows whose scores are NaN (a query that is not finite)
are NaN and change no other row, whatever the splits of their keys; rows
without keys are 0 whatever their queries; through the partial triples and
their combine too."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield


def _inputs(dt, lens, D):
    g = torch.Generator(device="cuda").manual_seed(len(lens) + D)
    ps, Hkv = 16, 2
    need = [-(-n // ps) for n in lens]
    kv = torch.randn(sum(need) + 1, ps, 2, Hkv, D, generator=g, device="cuda").to(DT[dt])
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    o = 0
    for b, k in enumerate(need):
        table[b, :k] = torch.arange(o, o + k)
        o += k
    q = torch.randn(len(lens), 8, D, generator=g, device="cuda").to(DT[dt])
    return q, kv[:, :, 0], kv[:, :, 1], table, torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("lens", [[8000, 31], [300 + i % 50 for i in range(400)], [64, 0, 5]])
def test_decode_queries_that_are_not_finite_reach_their_rows_alone(lens, dt, D):
    from kessie_b200 import ops
    q, k, v, table, sl = _inputs(dt, lens, D)
    want, parts = ops.paged_fog_decode(q, k, v, table, sl), torch.empty(2, *q.shape[:2], D + 2, device="cuda")
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[::2, 3] = bad[1::2, 6] = True
    q[::2, 3, 5] = float("nan")
    q[1::2, 6] = float("inf")                                         # scores of both signs: inf - inf
    keyless = sl == 0
    got = ops.paged_fog_decode(q, k, v, table, sl, out_partial=parts[0])
    seen = bad & ~keyless[:, None]
    assert got[seen].isnan().all() and torch.equal(got[~bad], want[~bad])
    assert got[keyless].count_nonzero() == 0
    # the combine of this shard and one without keys
    ops.paged_fog_decode(q, k, v, table, torch.zeros_like(sl), out_partial=parts[1])
    for order in (parts, parts.flip(0).contiguous()):
        joined = ops.lse_combine(order, out_dtype=torch.float32)
        assert joined[seen].isnan().all() and torch.isfinite(joined[~bad]).all()
        assert joined[keyless].count_nonzero() == 0
    assert ops.read_device_status() == 0
