"""GPU: calls of the scheduler-step operators at the edges of what they allow:
queries that are not finite, against the rule that a row's values reach that
row alone; the ends of int32 in the fog's boundary and sums of very many small
probabilities; plans that begin with whole tiles; the types' lowest values, all
against 64 bits; and the mixed steps of the vLLM attention."""

from types import SimpleNamespace

import pytest
import torch

from tests.test_gpu_step_ops import DT, _Case, _i32

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


# ------------------------------------------------------------------ many small probabilities
@pytest.mark.parametrize("fog", ["none", "values"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_chunks_many_small_probabilities_add_up(dt, fog):
    """One key takes nearly all of a row, 131,071 others e^-16.25 each: 1.1 % of
    the output together.  The chunk is long enough that a block goes through
    all keys of a tile in one piece, with the maximum from the first key tile.

    P is held in 16 bits: relative h, and in fp16 an absolute 2^-25 of the 2^7
    that the largest probability is held at, 2^-32 a key of the row's maximum.
    The scores are exact here (one product each); the exponent's fp32 rounding
    (2^-24 of 23) and the exponential are good to 1e-5."""
    from kessie_b200 import ops
    S, T, H, D, ps = 131072, 4864, 8, 64, 64
    pages = S // ps
    kv = torch.zeros(pages, ps, 2, H, D, dtype=DT[dt], device="cuda")
    kv[0, 0, 0, :, 0] = 16.25
    kv[:, :, 1] = 1.0
    kv[0, 0, 1] = 0.0
    q = torch.zeros(T, H, D, dtype=DT[dt], device="cuda")
    q[:, :, 0] = 8.0                                                  # score 8 * 16.25 / sqrt(64)
    clear = S // 2
    got = ops.paged_fog_chunks(q, kv[:, :, 0], kv[:, :, 1], torch.arange(pages, device="cuda").int()[None],
                               _i32([0, T]), _i32([S]), clear_start=_i32([clear]) if fog == "values" else None,
                               fog_alpha=0.5)
    j = torch.arange(S, dtype=torch.float64, device="cuda")
    w = torch.where(j < clear, (j / (clear - 1)).sqrt(), 1.0) if fog == "values" else torch.ones_like(j)
    w[0] = 0.0                                                        # that key's value
    p = torch.arange(S - T, S, device="cuda")
    small = torch.tensor(-16.25, dtype=torch.float64, device="cuda").exp()
    den = 1 + p * small
    want = (torch.cumsum(w, 0)[p] * small / den)[:, None, None]
    h = torch.finfo(DT[dt]).eps / 2
    tol = want * (2.01 * h + 2e-5) + (S * 2.0 ** -32 if dt == "fp16" else 0.0)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"worst {err.max().item()} at {want.min().item()} .. {want.max().item()}"


# ------------------------------------------------------------------ the vLLM attention's mixed steps
@pytest.fixture
def fog_on():
    from kessie_b200 import kessie_attention as A
    A.KESSIE_STATE.update(fog_alpha=1.5, fog_start=0.5, prompt_len=10, recall_positions=[], recall_boost=0.0)
    A.KESSIE_STATE.enabled = True
    yield A
    A.KESSIE_STATE.update(prompt_len=0)


class _Step:
    """A vLLM step of KeSSieAttentionImpl over a _Case's cache."""

    def __init__(self, A, c, **metadata):
        Hq, D = c.q.shape[1:]
        inner = SimpleNamespace(num_heads=Hq, num_kv_heads=c.k.shape[2], head_size=D, scale=D ** -0.5,
                                sliding_window=None)
        self.impl, self.c, self.cache = A.KeSSieAttentionImpl(_inner_impl=inner), c, torch.stack([c.k, c.v])
        self.md = SimpleNamespace(num_actual_tokens=sum(c.q_lens), max_query_len=max(c.q_lens),
                                  query_start_loc=c.start, seq_lens=c.seq, block_table=c.bt,
                                  max_seq_len=max(c.kv_lens), **metadata)
        self.out = torch.full((c.q.shape[0], Hq * D), 2.0, dtype=c.q.dtype, device="cuda")

    def forward(self):
        assert self.impl.forward(None, self.c.q, None, None, self.cache, self.md, self.out) is self.out
        return self.out.view(self.c.q.shape)


def test_vllm_mixed_step_refuses_a_length_past_the_block_table(fog_on):
    """As the call per request did: an error, not a device status bit that the
    attention never reads.  A bound above the table alone is no error."""
    c = _Case(74, [1, 60, 7], [900, 300, 77], 8, 2, 128, 16, "bf16", layout="vllm")
    step = _Step(fog_on, c)
    want = step.forward().clone()
    step.md.max_seq_len = 10 ** 6                                     # vLLM's bound: every length fits all the same
    assert torch.equal(step.forward(), want)
    c.seq[1] = step.md.max_seq_len = c.bt.shape[1] * 16 + 1
    with pytest.raises(ValueError, match="capacity"):
        step.forward()


def _fog_bias_16(dt, recalled=()):
    """kv_len -> the step's bias, rounded to the 16-bit type at each operation as torch rounds it."""
    r = lambda x: x.to(DT[dt]).float()

    def bias(s):
        j, fb = torch.arange(s, device="cuda"), int(s * 0.5)
        d = r(1.0 - r(r(j.float()) / max(fb, 1)))
        x = torch.where(j < fb, r(r(d * d) * -1.5), 0.0).double()
        for p in recalled:
            if p < s:
                x[p] = 0.25
        return x
    return bias


def test_vllm_mixed_step_of_more_sequences_than_one_call_takes(fog_on):
    from kessie_b200 import ops
    B = ops.MAX_CHUNK_SEQUENCES + 5
    q_lens = [1 if i % 100 else 3 for i in range(B)]
    q_lens[ops.MAX_CHUNK_SEQUENCES - 2:ops.MAX_CHUNK_SEQUENCES + 2] = [2, 40, 1, 70]     # around the border
    kv_lens = [n + i % 37 for i, n in enumerate(q_lens)]
    c = _Case(75, q_lens, kv_lens, 4, 1, 64, 16, "bf16", layout="vllm", pad=3)
    step = _Step(fog_on, c)
    got = step.forward()
    assert (got[sum(q_lens):] == 2.0).all()
    c.check(got, bias=_fog_bias_16("bf16"))


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("order", ["decodes first", "chunks first"])
def test_vllm_mixed_step_of_many_decodes(fog_on, monkeypatch, order, dt):
    """One run of decodes and one of chunks (requests without new tokens among
    them): a call of each, the rows of both as in the 64-bit run; the same step
    captured is one call, which holds for other lengths."""
    A = fog_on
    A.KESSIE_STATE.update(recall_positions=[3, 250, 700], recall_boost=0.25)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    Hkv = 8
    many = -(-3 * sms // Hkv) + 1
    decodes, chunks = [1] * many, [60, 0, 7, 200]
    q_lens = decodes + chunks if order == "decodes first" else chunks + decodes
    kv_lens = [n + 17 * i % 900 for i, n in enumerate(q_lens)]
    c = _Case(76, q_lens, kv_lens, 16, Hkv, 64, 16, dt, layout="vllm", pad=5)
    step = _Step(A, c, query_runs=A.query_runs(c.start.tolist()))
    calls = []
    for name in ("paged_fog_decode", "paged_fog_chunks"):
        def spy(*a, _f=getattr(A.ops, name), _name=name, **kw):
            calls.append(_name)
            return _f(*a, **kw)
        monkeypatch.setattr(A.ops, name, spy)
    bias = _fog_bias_16(dt, [3, 250, 700])
    got = step.forward()
    assert sorted(calls) == ["paged_fog_chunks", "paged_fog_decode"]
    assert (got[sum(q_lens):] == 2.0).all()
    c.check(got, bias=bias)
    del calls[:]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.forward()
    assert calls == ["paged_fog_chunks"]
    c.q_lens = q_lens[::-1]
    c.kv_lens = [max(s - 5, 0) for s in kv_lens]                      # some with fewer keys than new tokens
    c.start.copy_(_i32([sum(c.q_lens[:i]) for i in range(len(q_lens) + 1)]))
    c.seq.copy_(_i32(c.kv_lens))
    step.out.fill_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert (got[sum(q_lens):] == 2.0).all()
    c.check(got, bias=bias)


# ------------------------------------------------------------------ whole tiles first
def _whole_tiles(q_lens, kv_lens, Hq, Hkv, window=0, causal=True):
    """(whole tiles a block takes first, tiles left to cut, single tiles) of the
    plan, restated: tiles of 2 * (128 / G) tokens; a key tile of 128 costs 3
    (2 for a tile of one half) and a tile 7; whole tiles come first where a tile
    costs 192 or more in the mean and (sequence, head) has at least 2 tiles."""
    blocks = torch.cuda.get_device_properties(0).multi_processor_count
    half = 128 // (Hq // Hkv)
    cost = tiles = single = 0
    for n, s in zip(q_lens, kv_lens):
        for t0 in range(0, n, 2 * half):
            m = min(n - t0, 2 * half)
            first = s - n + t0
            hi = max(0, min(s, first + m)) if causal or window else s
            lo = min(max(first - window + 1, 0), hi) if window else 0
            keys = max(1, -(-hi // 128) - lo // 128)
            cost += Hkv * (keys * (2 if m <= half else 3) + 7)
            tiles += Hkv
            single += Hkv * (m <= half)
    whole = min(tiles // blocks, 128) if cost >= 192 * tiles and tiles >= 2 * len(q_lens) * Hkv else 0
    return whole, tiles - whole * blocks, single


# name: (new tokens, keys, Hq, Hkv, D, window, causal), with 148 blocks
WHOLE = {
    "one a block, a few cut": ([608], [20000], 64, 8, 64, 0, True),
    "one a block, none cut": ([1180], [20000], 32, 4, 128, 0, True),
    "two a block, most of a third cut": ([900, 750], [20000, 15000], 64, 8, 64, 0, True),
    "two a block, single tiles": ([700, 650, 8, 1], [20000, 30000, 9000, 12000], 64, 8, 64, 0, True),
    "window": ([700, 300], [24000, 20000], 64, 8, 128, 9000, True),
    "contexts far apart": ([300, 1200], [40000, 1200], 32, 8, 128, 0, True),
    "cross attention": ([400, 500], [16000, 9000], 64, 8, 64, 0, False)}


@pytest.mark.parametrize("fog", ["none", "values", "scores"])
@pytest.mark.parametrize("name", list(WHOLE))
def test_chunks_whole_tiles_first(name, fog):
    """Long contexts shared by many tiles: each block takes whole tiles before
    the rest is cut; into the queries themselves, too."""
    from kessie_b200 import ops
    q_lens, kv_lens, Hq, Hkv, D, window, causal = WHOLE[name]
    whole, left, single = _whole_tiles(q_lens, kv_lens, Hq, Hkv, window, causal)
    assert whole >= (2 if name.startswith("two") else 1), f"no case of whole tiles on this GPU: {whole}, {left}"
    assert (left == 0) == name.endswith("none cut") and (single > 8 or "single" not in name)
    c = _Case(77, q_lens, kv_lens, Hq, Hkv, D, 16, "fp16" if fog == "values" else "bf16")
    clear = [n * 3 // 4 for n in kv_lens] if fog == "values" else None
    kw = dict(window_size=window, causal=causal)
    bias = None
    if fog == "values":
        kw.update(clear_start=_i32(clear), fog_alpha=0.7)
    elif fog == "scores":
        kw.update(bias=ops.FogBias(1.5, 0.4, [3, 250, 8000], 0.25, dtype=torch.float32), fog_alpha=0.0)

        def bias(s):
            j, fb = torch.arange(s, device="cuda", dtype=torch.float64), int(s * 0.6)
            x = torch.where(j < fb, -1.5 * (1 - j / max(fb, 1)) ** 2, 0.0)
            for p in (3, 250, 8000):
                if p < s:
                    x[p] = 0.25
            return x
    got = c.run(**kw)
    c.check(got, clear=clear, alpha=0.7, window=window, causal=causal, bias=bias)
    assert torch.equal(c.run(**kw), got)
    assert c.run(out=c.q, **kw) is c.q and torch.equal(c.q, got)


# ------------------------------------------------------------------ the lowest values
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_chunks_values_of_the_types_lowest_value(dt):
    """A value row of the type's lowest value among others, under equal scores
    (all probabilities are 1, so that no sum leaves fp32)."""
    c = _Case(78, [1, 5, 40], [600, 70, 1200], 8, 2, 128, 16, dt, scale=0.0)
    for b in range(3):
        c.v[c.bt[b, 0], 0] = torch.finfo(DT[dt]).min
    c.check(c.run())
