"""GPU: the scheduler-step operators against plain implementations in 64 bits:
step tables (exact), multi-axis rotary with slot insert and remap, attention of
ragged chunks over the paged cache, and a step of all three, captured too.

Tolerances.  A rounding to the output type is off by at most h |o|, h =
finfo.eps / 2.  The attention also rounds each probability to the operands'
type (relative h, so h A with A = sum p w |v| / sum p; in fp16 a probability
below 2^-14 of the row's reference is subnormal, off by 2^-25 absolute).  The
scores are fp32 sums of D exact products: D 2^-23 sum |q_i k_i| scale, at the
inputs' sizes below 2e-4, entering numerator and denominator (4e-4 A); the
exponentials, fog weights and rescales are good to 1e-5.  For the rotary, the
angle is off by pi 2^-25 plus sincospif's 2 ulp and three fp32 roundings:
below 5e-7 (|x| + |y|) before the rounding to the stored type."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield


@pytest.fixture(autouse=True)
def _status():
    from kessie_b200 import ops
    ops.read_device_status()
    yield
    assert ops.read_device_status() == 0, "device status bits left by a test that expects none"


def _half_eps(dt):
    return torch.finfo(DT[dt]).eps / 2


def _i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ step tables
def _tables_plain(ctx, new, table, ps, free, num_tokens):
    table = table.copy()
    free = list(free)
    used, start, pos, slots = 0, [0], [], []
    for r, (c, n) in enumerate(zip(ctx, new)):
        for p in range(-(-c // ps), -(-(c + n) // ps)):
            table[r, p] = free.pop()
            used += 1
        for t in range(n):
            pos.append(c + t)
            slots.append(int(table[r, (c + t) // ps]) * ps + (c + t) % ps)
        start.append(start[-1] + n)
    pad = num_tokens - len(pos)
    return start, [c + n for c, n in zip(ctx, new)], pos + [0] * pad, slots + [-1] * pad, used, table


def _tables_inputs(seed, ctx, new, ps, extra_width=0, extra_free=3):
    rng = np.random.default_rng(seed)
    owned = [-(-c // ps) for c in ctx]
    need = [-(-(c + n) // ps) for c, n in zip(ctx, new)]
    pool = sum(need) + extra_free
    perm = rng.permutation(pool).astype(np.int32)
    table = np.full((len(ctx), max(need + [1]) + extra_width), -7, np.int32)
    o = 0
    for r, k in enumerate(owned):
        table[r, :k] = perm[o:o + k]
        o += k
    return table, perm[o:], pool


@pytest.mark.parametrize("ps", [1, 16, 48])
@pytest.mark.parametrize("ctx,new,pad", [
    ([0], [1], 0), ([5], [0], 2), ([15, 16, 17, 0], [1, 1, 1, 1], 0), ([0, 0, 7, 31], [0, 100, 0, 1], 5),
    ([1000, 3, 0, 47, 48], [33, 0, 0, 2, 500], 11), ([0, 0, 0], [0, 0, 0], 4)])
def test_step_tables(ps, ctx, new, pad):
    from kessie_b200 import ops
    table, free, pool = _tables_inputs(len(ctx) + pad, ctx, new, ps, extra_width=2)
    want = _tables_plain(ctx, new, table, ps, free, sum(new) + pad)
    # a table that is a view of a wider one: the rest of each row stays
    wide = torch.full((len(ctx), table.shape[1] + 3), 99, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = torch.from_numpy(table)
    dev = wide[:, :table.shape[1]]
    got = ops.step_tables(_i32(ctx), _i32(new), dev, ps, torch.from_numpy(free.copy()).cuda(), sum(new) + pad,
                          num_pages=pool)
    assert got.query_start_loc.tolist() == want[0] and got.seq_lens.tolist() == want[1]
    assert got.positions.tolist() == want[2] and got.slot_mapping.tolist() == want[3]
    assert got.pages_used.item() == want[4]
    np.testing.assert_array_equal(dev.cpu().numpy(), want[5])
    assert (wide[:, table.shape[1]:] == 99).all()


@pytest.mark.parametrize("R", [1, 1023, 1025, 5000, 8192])
def test_step_tables_many_requests(R):
    from kessie_b200 import ops
    rng = np.random.default_rng(R)
    ctx = rng.integers(0, 200, R).tolist()
    new = (rng.integers(0, 40, R) * (rng.random(R) < 0.5)).tolist()
    table, free, pool = _tables_inputs(R, ctx, new, 16)
    want = _tables_plain(ctx, new, table, 16, free, sum(new) + 1)
    dev = torch.from_numpy(table.copy()).cuda()
    got = ops.step_tables(_i32(ctx), _i32(new), dev, 16, torch.from_numpy(free.copy()).cuda(), sum(new) + 1)
    assert got.query_start_loc.tolist() == want[0] and got.positions.tolist() == want[2]
    assert got.slot_mapping.tolist() == want[3] and got.pages_used.item() == want[4]
    np.testing.assert_array_equal(dev.cpu().numpy(), want[5])


def test_step_tables_free_count_int64_lengths_and_reused_outputs():
    from kessie_b200 import ops
    ctx, new = [10, 0], [10, 5]
    table, free, pool = _tables_inputs(3, ctx, new, 16, extra_free=0)
    longer = np.concatenate([free, np.array([1000, 1001], np.int32)])       # entries past free_count are not free
    want = _tables_plain(ctx, new, table, 16, free, 15)
    dev = torch.from_numpy(table.copy()).cuda()
    count = _i32([len(free)])
    lens = (torch.tensor(ctx, device="cuda"), torch.tensor(new, device="cuda"))
    a = ops.step_tables(*lens, dev, 16, torch.from_numpy(longer).cuda(), 15, num_pages=pool, free_count=count)
    b = ops.step_tables(*lens, dev, 16, torch.from_numpy(longer).cuda(), 15, num_pages=pool, free_count=count, out=a)
    assert b.slot_mapping.data_ptr() == a.slot_mapping.data_ptr() and b.slot_mapping.tolist() == want[3]
    assert count.item() == len(free) and b.pages_used.item() == want[4]


def test_step_tables_without_requests_or_tokens():
    from kessie_b200 import ops
    none = _i32([])
    got = ops.step_tables(none, none, torch.empty(0, 4, dtype=torch.int32, device="cuda"), 16, _i32([1, 2]), 3)
    assert got.query_start_loc.tolist() == [0] and got.slot_mapping.tolist() == [-1] * 3 and got.pages_used.item() == 0
    table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    got = ops.step_tables(_i32([3]), _i32([0]), table, 16, none, 0)          # no new token, no free page
    assert got.query_start_loc.tolist() == [0, 0] and got.seq_lens.tolist() == [3] and (table == -1).all()


def test_step_tables_far_slots_pass_32_bits():
    from kessie_b200 import ops
    table = torch.tensor([[200_000_000, -1]], dtype=torch.int32, device="cuda")
    got = ops.step_tables(_i32([15]), _i32([3]), table, 16, _i32([7, 210_000_000]), 3)
    assert got.slot_mapping.tolist() == [200_000_000 * 16 + 15, 210_000_000 * 16, 210_000_000 * 16 + 1]


def test_step_tables_records_what_does_not_fit():
    from kessie_b200 import _lib, ops
    free = _i32([4, 5])
    table = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    got = ops.step_tables(_i32([0, 0]), _i32([33, 4]), table, 16, free, 37, num_pages=10)   # 33 tokens: 3 pages of 2
    assert ops.read_device_status() == _lib.DEV_BAD_ARG
    assert table[0].tolist() == [5, 4] and table[1].tolist() == [-1, -1]
    assert got.slot_mapping.tolist() == [80 + i for i in range(16)] + [64 + i for i in range(16)] + [-1] * 5
    assert got.pages_used.item() == 2
    table.fill_(-1)
    got = ops.step_tables(_i32([-3, 0]), _i32([2, -1]), table, 16, free, 1, num_pages=10)   # negative; one row too few
    assert ops.read_device_status() == _lib.DEV_BAD_ARG
    assert got.query_start_loc.tolist() == [0, 2, 2] and got.seq_lens.tolist() == [2, 0]
    assert got.positions.tolist() == [0]
    table = torch.tensor([[3, -1]], dtype=torch.int32, device="cuda")
    got = ops.step_tables(_i32([4]), _i32([2]), table, 16, free, 2, num_pages=3)            # page 3 of 3
    assert ops.read_device_status() == _lib.DEV_BAD_PAGE_ID and got.slot_mapping.tolist() == [-1, -1]
    with pytest.raises(ValueError, match="int32"):
        ops.step_tables(_i32([4]), _i32([2]), table.long(), 16, free, 2)
    with pytest.raises(ValueError, match="one context"):
        ops.step_tables(_i32([4, 5]), _i32([2, 1]), table, 16, free, 2)


# ------------------------------------------------------------------ rotary
def _axis_of(sections, interleaved):
    A = len(sections)
    if interleaved:
        return [d % A if d < A * sections[d % A] else 0 for d in range(sum(sections))]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def _rotate64(x, delta, sections, theta, interleaved):
    """float64 rotation of x [T, H, D] by delta [A, T], and |x| + |y| of each element's pair."""
    half = sum(sections)
    f = np.array([theta ** (-d / half) for d in range(half)]).astype(np.float32).astype(np.float64)
    ang = delta[_axis_of(sections, interleaved)].T.astype(np.float64) * f                # [T, half]
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    x = x.double().cpu().numpy()
    a, b = x[..., :half], x[..., half:2 * half]
    both = np.abs(a) + np.abs(b)
    return (np.concatenate([a * c - b * s, a * s + b * c, x[..., 2 * half:]], -1),
            np.concatenate([both, both, np.zeros_like(x[..., 2 * half:])], -1))


def _assert_rotated(got, want, both, dt):
    err = np.abs(got.double().cpu().numpy() - want)
    tol = _half_eps(dt) * (np.abs(want) + 5e-7 * both) + 5e-7 * both
    if dt == "fp16":
        tol += 2.0 ** -25                                                                # subnormal results
    assert (err <= tol).all(), f"worst excess {np.max(err - tol)} at {np.unravel_index(np.argmax(err - tol), err.shape)}"


ROPE_CASES = [  # T, H, D, sections, interleaved, theta
    (1, 1, 128, (64,), False, 1e4), (7, 5, 128, (16, 24, 24), False, 1e6), (33, 3, 64, (12, 10, 10), True, 5e5),
    (5, 2, 96, (10, 6), False, 1e4), (300, 8, 128, (24, 20, 20), True, 5e6), (3, 40, 64, (3, 0, 13), False, 1e4),
    (9, 2, 80, (40,), False, 1e4), (4, 3, 20, (4, 3, 3), True, 1e4), (2, 2, 256, (32, 32, 32, 32), False, 1e4),
    (2, 1, 512, (256,), False, 1e4)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H,D,sections,inter,theta", ROPE_CASES)
def test_rope_axes_remap(dt, T, H, D, sections, inter, theta):
    from kessie_b200 import ops
    g = torch.Generator().manual_seed(T * D + H)
    A = len(sections)
    k = torch.randn(T, H, D, generator=g).to(DT[dt]).cuda()
    # signed, far and equal positions
    org = torch.randint(-(1 << 20), 1 << 20, (A, T), generator=g, dtype=torch.int32)
    tgt = torch.randint(0, 1 << 20, (A, T), generator=g, dtype=torch.int32)
    tgt[0, 0] = org[0, 0]
    want, both = _rotate64(k, (tgt.long() - org.long()).numpy(), sections, theta, inter)
    out = torch.empty_like(k)
    assert ops.rope_axes_remap(k, org.cuda(), tgt.cuda(), sections, theta, inter, out=out) is out
    _assert_rotated(out, want, both, dt)
    same = ops.rope_axes_remap(k, org.cuda(), tgt.cuda(), sections, theta, inter)        # in place
    assert same is k and torch.equal(k, out)


def test_rope_axes_remap_extreme_positions_strides_and_int64():
    """int32's ends, rows inside a wider tensor, unaligned rows (the element-wise
    form), positions as a strided int64 view."""
    from kessie_b200 import ops
    sections = (16, 24, 24)
    tgt = torch.tensor([[2 ** 31 - 1, 0], [0, -2 ** 31], [5, 2 ** 31 - 1]])
    org = torch.tensor([[-2 ** 31, 0], [2 ** 31 - 1, 2 ** 31 - 1], [5, 0]])
    wide = torch.randn(2, 3, 131, generator=torch.Generator().manual_seed(1)).cuda()
    for x in (wide[:, :, :128], wide[:, :, 3:]):
        want, both = _rotate64(x, (tgt - org).numpy(), sections, 1e4, False)
        out = torch.empty(2, 3, 128, device="cuda")
        strided = torch.stack([tgt, tgt], -1).cuda()[..., 0]
        ops.rope_axes_remap(x, org.cuda(), strided, sections, 1e4, out=out)
        _assert_rotated(out, want, both, "fp32")


def test_rope_axes_remap_one_axis_agrees_with_rope_remap():
    from kessie_b200 import ops
    k = torch.randn(50, 4, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    org, tgt = torch.arange(50, dtype=torch.int32).cuda(), (torch.arange(50, dtype=torch.int32) * 3 + 100).cuda()
    a = ops.rope_axes_remap(k.clone(), org, tgt, [64], 5e5)
    b = ops.rope_remap(k.clone(), org, tgt, 5e5)
    # the one-axis remap rounds its angle (at most 250 here) to fp32: 1.5e-5
    assert ((a.float() - b.float()).abs() <= 2 * _half_eps("bf16") * b.float().abs() + 1e-4).all()


@pytest.mark.parametrize("layout", ["kessie", "vllm"])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,Hq,Hkv,D,ps,sections,inter", [
    (1, 8, 2, 128, 16, (64,), False), (45, 32, 8, 128, 16, (16, 24, 24), False), (700, 6, 2, 64, 32, (8, 8), False),
    (19, 3, 1, 96, 5, (24, 12, 12), True), (6, 4, 4, 20, 16, (10,), False)])
def test_rope_axes_insert(layout, dt, T, Hq, Hkv, D, ps, sections, inter):
    from kessie_b200 import ops
    g = torch.Generator().manual_seed(T + D)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g).to(DT[dt]).cuda()
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    P = -(-T // ps) + 2
    shape = (P, ps, 2, Hkv, D) if layout == "kessie" else (2, P, ps, Hkv, D)
    kv = torch.full(shape, 7.0, dtype=DT[dt], device="cuda")
    pos = torch.randint(0, 300000, (len(sections), T), generator=g, dtype=torch.int32)
    slots = torch.randperm(P * ps, generator=g)[:T]
    if T > 2:
        slots[1] = -1                                                 # a padded row
    wq, bq = _rotate64(q, pos.numpy(), sections, 1e6, inter)
    wk, bk = _rotate64(k, pos.numpy(), sections, 1e6, inter)
    out = ops.rope_axes_insert(q, k, v, pos.cuda(), sections, kv, slots.cuda(), 1e6, inter,
                               out_q=torch.empty(T, Hq, D, dtype=DT[dt], device="cuda"), layout=layout)
    _assert_rotated(out, wq, bq, dt)
    rows = (kv if layout == "vllm" else kv.permute(2, 0, 1, 3, 4)).reshape(2, P * ps, Hkv, D)
    live = slots >= 0
    _assert_rotated(rows[0][slots[live]], wk[live.numpy()], bk[live.numpy()], dt)
    assert torch.equal(rows[1][slots[live]], v[live.cuda()])
    rest = torch.ones(P * ps, dtype=torch.bool)
    rest[slots[live]] = False
    assert (rows[:, rest.cuda()] == 7.0).all()                        # every other row is as it was
    ops.rope_axes_insert(q, k, v, pos.cuda(), sections, kv, slots.int().cuda(), 1e6, inter, layout=layout)
    assert torch.equal(q, out)                                        # in place, int32 slots


def test_rope_axes_insert_records_a_slot_past_the_cache():
    from kessie_b200 import _lib, ops
    x = torch.randn(3, 2, 64, device="cuda")
    kv = torch.zeros(2, 16, 2, 2, 64, device="cuda")
    pos = torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    ops.rope_axes_insert(x, x, x, pos, [32], kv, torch.tensor([32, 1, 1 << 40], device="cuda"))
    assert ops.read_device_status() == _lib.DEV_BAD_PAGE_ID
    assert torch.equal(kv[0, 1, 0], x[1]) and kv.count_nonzero() == 2 * x[1].count_nonzero()
    with pytest.raises(ValueError, match="positions"):
        ops.rope_axes_insert(x, x, x, pos[:, :2], [32], kv, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError, match="dtype"):
        ops.rope_axes_insert(x.half(), x, x, pos, [32], kv, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="cache of"):
        ops.rope_axes_insert(x, x[:, :1], x[:, :1], pos, [32], kv, torch.zeros(3, dtype=torch.int64, device="cuda"))


# ------------------------------------------------------------------ ragged chunks
class _Case:
    """Seeded inputs of a ragged batch over a randomly placed cache."""

    def __init__(self, seed, q_lens, kv_lens, Hq, Hkv, D, ps, dt, layout="kessie", pad=0, scale=1.5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_lens, self.kv_lens, self.dt, self.ps, self.D = q_lens, kv_lens, dt, ps, D
        need = [-(-n // ps) for n in kv_lens]
        P = sum(need) + 2
        shape = {"kessie": (P, ps, 2, Hkv, D), "vllm": (2, P, ps, Hkv, D), "heads": (P, 2, Hkv, ps, D),
                 "odd": (P, ps, 2, Hkv, D + 8)}[layout]
        kv = torch.randn(shape, generator=g, device="cuda").to(DT[dt])
        if layout == "vllm":
            self.k, self.v = kv[0], kv[1]
        elif layout == "heads":                                       # [P, 2, H, ps, D]: tokens inside heads
            self.k, self.v = kv[:, 0].transpose(1, 2), kv[:, 1].transpose(1, 2)
        else:
            self.k, self.v = kv[:, :, 0, :, :D], kv[:, :, 1, :, :D]
        perm = torch.randperm(P, generator=g, device="cuda").int()
        self.bt = torch.full((len(kv_lens), max(need + [1])), -1, dtype=torch.int32, device="cuda")
        o = 0
        for b, n in enumerate(need):
            self.bt[b, :n] = perm[o:o + n]
            o += n
        self.q = (torch.randn(sum(q_lens) + pad, Hq, D, generator=g, device="cuda") * scale).to(DT[dt])
        self.start = _i32(np.concatenate([[0], np.cumsum(q_lens)]))
        self.seq = _i32(kv_lens)

    def run(self, **kw):
        from kessie_b200 import ops
        return ops.paged_fog_chunks(self.q, self.k, self.v, self.bt, self.start, self.seq, **kw)

    def check(self, got, clear=None, alpha=0.5, window=0, causal=True, bias=None):
        """Compare with the 64-bit rows; bias: function kv_len -> float64 bias of each key."""
        h, row = _half_eps(self.dt), 0
        Hq, D = self.q.shape[1:]
        Hkv = self.k.shape[2]
        assert torch.isfinite(got[:sum(self.q_lens)]).all()
        for b, (n, s) in enumerate(zip(self.q_lens, self.kv_lens)):
            if n == 0:
                continue
            q = self.q[row:row + n].double().transpose(0, 1)                              # [Hq, n, D]
            ids = self.bt[b, :-(-s // self.ps)].long()
            k, v = ((c[ids].reshape(-1, Hkv, D)[:s].double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1))
                    for c in (self.k, self.v))
            j = torch.arange(s, device="cuda", dtype=torch.float64)
            p = torch.arange(n, device="cuda", dtype=torch.float64) + (s - n)
            gap = p[:, None] - j[None]
            seen = torch.ones_like(gap, dtype=torch.bool)
            if causal or window:
                seen &= gap >= 0
            if window:
                seen &= gap < window
            x = q @ k.transpose(1, 2) / math.sqrt(D)
            if bias is not None:
                x = x + bias(s)
            x = x.masked_fill(~seen, -math.inf)
            top = x.amax(-1, keepdim=True) if s else x.new_zeros(Hq, n, 1)
            e = torch.exp(x - torch.where(top.isinf(), 0.0, top))
            l = e.sum(-1, keepdim=True)
            if clear is not None:
                cs = int(clear[b])
                w = torch.ones(s, dtype=torch.float64, device="cuda")
                w[:max(cs, 0)] = (j[:max(cs, 0)] / max(cs - 1, 1)) ** alpha
                v = v * w[:, None]
            den = torch.where(l > 0, l, 1.0)
            want, mass = e @ v / den, e @ v.abs() / den
            if s:
                sub = s * 2.0 ** -25 * v.abs().amax(1, keepdim=True) / den if self.dt == "fp16" else 0.0
            else:
                sub = 0.0
            tol = h * (want.abs() + 1.01 * mass) + 4.2e-4 * mass + sub + 1e-30
            err = (got[row:row + n].double().transpose(0, 1) - want).abs()
            worst = (err - tol).max().item()
            assert worst <= 0, f"sequence {b} (n {n}, s {s}): error exceeds the bound by {worst}"
            row += n


LENGTHS = [
    ([1], [1]), ([1], [129]), ([3], [3]), ([1, 1, 1, 1], [5, 300, 128, 4000]), ([64, 1, 17, 130], [64, 777, 2000, 131]),
    ([0, 5, 0, 1, 0], [40, 5, 0, 0, 700]), ([300], [900]), ([33, 600, 2], [1500, 601, 5000])]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (6, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("q_lens,kv_lens", LENGTHS)
def test_chunks(dt, Hq, Hkv, D, q_lens, kv_lens):
    c = _Case(sum(kv_lens) + Hq, q_lens, kv_lens, Hq, Hkv, D, 16, dt)
    c.check(c.run())


@pytest.mark.parametrize("q_lens,kv_lens", LENGTHS)
def test_chunks_value_fog(q_lens, kv_lens):
    c = _Case(3, q_lens, kv_lens, 8, 2, 128, 32, "bf16")
    clear = [n * 3 // 4 for n in kv_lens]
    c.check(c.run(clear_start=_i32(clear), fog_alpha=0.7), clear=clear, alpha=0.7)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [1, 100, 128, 1000])
def test_chunks_window(window, D):
    c = _Case(window, [1, 40, 300, 2], [3000, 1500, 300, 90], 8, 4, D, 16, "fp16")
    c.check(c.run(window_size=window), window=window)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_chunks_score_fog_and_recall(dt):
    from kessie_b200 import ops
    c = _Case(9, [1, 70, 1], [2000, 500, 33], 8, 2, 128, 16, dt)
    recalled = [3, 250, 1999, 5000]

    def bias(s):
        j = torch.arange(s, device="cuda", dtype=torch.float64)
        fb = int(s * 0.6)
        x = torch.where(j < fb, -1.5 * (1 - j / max(fb, 1)) ** 2, 0.0)
        for r in recalled:
            if r < s:
                x[r] = 0.25
        return x
    c.check(c.run(bias=ops.FogBias(1.5, 0.4, recalled, 0.25, dtype=torch.float32), fog_alpha=0.0), bias=bias)


@pytest.mark.parametrize("layout,ps", [("vllm", 16), ("heads", 16), ("odd", 32), ("kessie", 48), ("kessie", 128),
                                       ("vllm", 256), ("heads", 80)])
@pytest.mark.parametrize("D", [64, 128])
def test_chunks_layouts_and_page_sizes(layout, ps, D):
    c = _Case(ps, [1, 50, 200], [1000, 777, 201], 8, 2, D, ps, "bf16", layout=layout)
    c.check(c.run())


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 1), (64, 8), (7, 7), (128, 1), (100, 2)])
def test_chunks_head_groups(Hq, Hkv):
    c = _Case(Hq, [1, 9, 140], [400, 350, 1300], Hq, Hkv, 128, 16, "bf16")
    c.check(c.run())


@pytest.mark.parametrize("q_lens,kv_lens", [([5, 1, 200], [700, 1, 50]), ([300], [0]), ([17], [100000])])
def test_chunks_cross_attention(q_lens, kv_lens):
    """Not causal: every row sees all keys of a sequence of another length."""
    c = _Case(5, q_lens, kv_lens, 8, 2, 128, 16, "fp16")
    c.check(c.run(causal=False), causal=False)


def test_chunks_rows_without_keys_are_zero():
    """A sequence with fewer keys than queries: its first rows sit before key 0."""
    c = _Case(6, [200, 3], [50, 0], 8, 2, 128, 16, "bf16")
    out = c.run(out=torch.full_like(c.q, 9.0))
    assert out[:150].count_nonzero() == 0 and out[200:].count_nonzero() == 0
    c.check(out)


def test_chunks_padded_rows_stay_and_unused_keys_hold_anything():
    """Rows behind the last sequence keep their contents; NaN behind the last
    key of a page, on pages before the window, and in the rows' own padding."""
    c = _Case(7, [1, 40], [500, 300], 8, 2, 128, 16, "bf16", pad=9)
    c.q[41:] = float("nan")
    c.k[c.bt[0, 500 // 16], 500 % 16:] = float("nan")
    c.v[c.bt[0, 500 // 16], 500 % 16:] = float("inf")
    c.v[c.bt[1, 300 // 16], 300 % 16:] = float("nan")
    out = torch.full_like(c.q, 3.0)
    got = c.run(out=out)
    assert got is out and (out[41:] == 3.0).all()
    c.check(out)
    # window 64: keys 0 .. 299 - 40 - 64 of sequence 1 and 0 .. 435 of sequence 0 are seen by no row
    c.k[c.bt[0, :27]] = float("nan")
    c.v[c.bt[0, :27]] = float("nan")
    c.v[c.bt[0, 27], :4] = float("-inf")
    c.v[c.bt[1, :12]] = float("nan")
    clean = _Case(7, [1, 40], [500, 300], 8, 2, 128, 16, "bf16", pad=9)
    got = c.run(window_size=64, out=out)
    clean.check(got, window=64)


def test_chunks_masked_pages_may_be_missing():
    """Page ids before the window or behind the last key are not looked at."""
    c = _Case(8, [1, 30], [900, 640], 8, 2, 128, 16, "bf16")
    want = c.run(window_size=100)
    c.bt[0, :48] = -1
    c.bt[1, :30] = 1 << 30
    c.bt = torch.cat([c.bt, torch.full((2, 5), -9, dtype=torch.int32, device="cuda")], 1)
    assert torch.equal(c.run(window_size=100), want)


def test_chunks_bad_page_and_lengths_are_recorded():
    from kessie_b200 import _lib, ops
    c = _Case(8, [1, 30], [900, 640], 8, 2, 128, 16, "bf16")
    c.bt[0, 3] = c.k.shape[0]
    out = c.run()
    assert ops.read_device_status() == _lib.DEV_BAD_PAGE_ID and torch.isfinite(out).all()
    c = _Case(8, [1, 30], [900, 640], 8, 2, 128, 16, "bf16")
    c.run(max_seq_len=800)
    assert ops.read_device_status() == _lib.DEV_BAD_ARG
    c.start = _i32([0, 1, 77])                                        # past the rows of q
    c.run()
    assert ops.read_device_status() == _lib.DEV_BAD_ARG
    c.start = _i32([5, 2, 31])                                        # falling
    c.run()
    assert ops.read_device_status() == _lib.DEV_BAD_ARG
    with pytest.raises(ValueError, match="capacity"):
        c.run(max_seq_len=10 ** 6)
    with pytest.raises(ValueError, match="query_start_loc"):
        ops.paged_fog_chunks(c.q, c.k, c.v, c.bt, c.start[:2], c.seq)


def test_chunks_strided_and_unaligned_queries():
    """q inside a fused qkv tensor, q at an odd element offset (copied), out inside a wider tensor."""
    c = _Case(4, [1, 20], [300, 400], 8, 2, 128, 16, "bf16")
    want = c.run()
    qkv = torch.randn(21, 12, 128, device="cuda").to(torch.bfloat16)
    qkv[:, :8] = c.q
    plain, c.q = c.q, qkv[:, :8]
    wide = torch.zeros(21, 10, 128, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(c.run(out=wide[:, 1:9]), want) and wide[:, 0].count_nonzero() == 0
    flat = torch.zeros(21 * 8 * 128 + 1, dtype=torch.bfloat16, device="cuda")
    c.q = flat[1:].view(21, 8, 128).copy_(plain)
    assert torch.equal(c.run(), want)
    with pytest.raises(Exception, match="aligned"):
        c.run(out=flat[1:].view(21, 8, 128))


def test_chunks_large_scores_and_lowest_values():
    """Scores far apart (one key takes all), and rows of the type's lowest value."""
    c = _Case(11, [1, 5, 40], [600, 70, 1200], 8, 2, 128, 16, "bf16", scale=0.0)
    c.q.fill_(1.0)
    c.k[c.bt[0, 5], 3] = 30.0                                         # score 339 against noise
    c.check(c.run())
    low = torch.finfo(torch.bfloat16).min
    c.q.zero_()
    c.v[c.bt[1, 0], 0] = low / 128
    got = c.run()
    assert torch.isfinite(got).all()


def test_chunks_far_offsets_pass_32_bits():
    """Pages whose element offset is past 2^31 (a cache of more than 4 GB)."""
    ps, H, D = 16, 8, 128
    pages = (1 << 31) // (ps * 2 * H * D) + 40
    kv = torch.zeros(pages, ps, 2, H, D, dtype=torch.bfloat16, device="cuda")
    c = _Case(12, [1, 30], [300, 200], 16, 8, 128, ps, "bf16")
    far = torch.arange(pages - c.k.shape[0], pages, device="cuda")
    kv[far, :, 0], kv[far, :, 1] = c.k, c.v
    want = c.run()
    c.bt = torch.where(c.bt >= 0, c.bt + int(far[0]), c.bt)
    c.k, c.v = kv[:, :, 0], kv[:, :, 1]
    assert torch.equal(c.run(), want)


def test_chunks_repeat_bit_for_bit_and_streams_do_not_share_scratch():
    from kessie_b200 import ops
    a = _Case(21, [1, 7, 33], [30000, 9000, 20000], 8, 1, 128, 16, "bf16")
    b = _Case(22, [16, 1], [25000, 12000], 8, 1, 128, 16, "bf16")
    wa, wb = a.run(), b.run()
    assert all(torch.equal(a.run(), wa) for _ in range(5))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            got.append((a.run(), wa))
        got.append((b.run(out=torch.empty_like(wb), stream=s2), wb))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)
    assert ops.chunks_workspace_bytes(8, 1, 128) > 0


def test_chunks_two_captured_graphs_replayed_at_once():
    a = _Case(23, [1, 7, 33], [30000, 9000, 20000], 8, 1, 128, 16, "bf16")
    b = _Case(24, [16, 1], [25000, 12000], 8, 1, 128, 16, "bf16")
    wa, wb = a.run(), b.run()
    oa, ob = torch.empty_like(wa), torch.empty_like(wb)
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        a.run(out=oa)
    with torch.cuda.graph(gb):
        b.run(out=ob)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        oa.zero_(), ob.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(s1):
                ga.replay()
            with torch.cuda.stream(s2):
                gb.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa, wa) and torch.equal(ob, wb)
    # other lengths, the same graph: the plan is made on the device
    a.seq.copy_(_i32([500, 8, 20000]))
    ga.replay()
    torch.cuda.synchronize()
    a.kv_lens = [500, 8, 20000]
    a.check(oa)


def test_chunks_from_two_host_threads_on_one_stream():
    """The kernel and its merge stay together, whoever else launches there."""
    import threading
    stream = torch.cuda.Stream()
    cases = [_Case(25, [1, 7, 33], [30000, 9000, 20000], 8, 1, 128, 16, "bf16"),
             _Case(26, [16, 1], [25000, 12000], 8, 1, 128, 16, "bf16")]
    want = [c.run() for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(stream):
            for _ in range(40):
                got[i].append(cases[i].run())
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_chunks_broadcast_queries_empty_batch_and_workspace():
    from kessie_b200 import ops
    c = _Case(27, [3, 2], [300, 200], 8, 2, 64, 16, "bf16")
    c.q = c.q[:1].expand(5, 8, 64)                                    # one query row for all tokens (stride 0)
    c.check(c.run())
    ws = torch.empty(ops.chunks_workspace_bytes(8, 2, 64), dtype=torch.uint8, device="cuda").fill_(255)
    assert torch.equal(c.run(ws=ws), c.run())                         # leftover contents are never read
    with pytest.raises(Exception, match="workspace"):
        c.run(ws=ws[:-16])
    empty = ops.paged_fog_chunks(c.q[:0], c.k, c.v, c.bt, c.start, c.seq)
    assert empty.shape == (0, 8, 64)
    with pytest.raises(Exception, match="not both"):
        c.run(clear_start=_i32([5, 5]), bias=ops.FogBias(1.0, 0.5, dtype=torch.float32))


def test_chunks_output_over_the_queries_and_falling_starts():
    for q_lens, kv_lens in (([1, 7, 33], [30000, 9000, 20000]), ([300, 2, 1], [900, 130, 64])):
        c = _Case(28, q_lens, kv_lens, 8, 1, 128, 16, "bf16")
        want = c.run()
        assert c.run(out=c.q) is c.q and torch.equal(c.q, want)
    from kessie_b200 import _lib, ops
    c.start = _i32([0, 300, 1, 303])
    out = torch.full_like(want, 7.0)
    c.run(out=out)
    assert ops.read_device_status() == _lib.DEV_BAD_ARG and (out == 7.0).all()
    with pytest.raises(Exception, match="share memory"):
        c.run(out=out[:1].expand_as(out))


@pytest.mark.parametrize("window", [140, 150, 2 ** 31 - 1])
def test_chunks_window_wider_than_the_sequences(window):
    """No less than causal attention, with more queries than keys too."""
    c = _Case(29, [200, 3], [140, 130], 8, 2, 128, 16, "bf16")
    want = c.run()
    c.check(want)
    for causal in (True, False):
        assert torch.equal(c.run(window_size=window, causal=causal, max_seq_len=140), want)


def test_conversions_run_on_the_given_stream():
    """64-bit lengths, positions and slots and an unaligned q are converted in
    the given stream's order, not behind the work of the current one."""
    from kessie_b200 import ops
    c = _Case(30, [1, 20], [300, 400], 8, 2, 128, 16, "bf16")
    want = c.run()
    flat = torch.zeros(21 * 8 * 128 + 1, dtype=torch.bfloat16, device="cuda")
    c.q = flat[1:].view(21, 8, 128).copy_(c.q)
    c.start, c.seq, c.bt = c.start.long(), c.seq.long(), c.bt.long()
    k = torch.randn(21, 2, 128, device="cuda")
    pos = torch.arange(63, device="cuda").view(3, 21)
    turned = ops.rope_axes_remap(k, None, pos, [16, 24, 24], out=torch.empty_like(k))
    R = 2
    free, table = torch.arange(40, device="cuda"), torch.full((R, 30), -1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([5, 40], device="cuda")
    tables = ops.step_tables(torch.zeros_like(lens), lens, table.clone(), 16, free, 45)
    zeros = torch.zeros_like(lens)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(400_000_000)                                    # the current stream is busy for a while
    busy.record()
    got = c.run(stream=s)
    gk = ops.rope_axes_remap(k, None, pos, [16, 24, 24], out=torch.empty_like(k), stream=s.cuda_stream)
    gt = ops.step_tables(zeros, lens, table, 16, free, 45, stream=s)
    s.synchronize()
    assert not busy.query()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(gk, turned)
    assert all(torch.equal(a, b) for a, b in zip(gt, tables))


# ------------------------------------------------------------------ a step of all three
@pytest.mark.parametrize("captured", [False, True])
def test_step_of_all_three(captured):
    """Two steps of four conversations (prompt chunks, then a mixed step):
    tables -> rotary + insert -> attention, against a dense 64-bit run over the
    tokens so far; the second step padded and, when captured, replayed."""
    from kessie_b200 import ops
    Hq, Hkv, D, ps, sections, theta = 8, 2, 128, 16, (16, 24, 24), 1e4
    g = torch.Generator(device="cuda").manual_seed(31)
    R, P = 4, 80
    kv = torch.full((P, ps, 2, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    table = torch.full((R, 20), -1, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(P, generator=g, device="cuda").int(), _i32([P])
    ctx = _i32([0] * R)
    hist = [[], [], [], []]
    for step, (new, pad) in enumerate([([200, 37, 0, 5], 0), ([1, 60, 130, 1], 8)]):
        T = sum(new) + pad
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device="cuda").to(torch.bfloat16)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        axes = torch.randint(0, 500, (2, T), generator=g, device="cuda", dtype=torch.int32)
        out, oq = torch.full((T, Hq, D), 5.0, dtype=torch.bfloat16, device="cuda"), torch.empty_like(q).contiguous()
        n = _i32(new)

        def run():
            t = ops.step_tables(ctx, n, table, ps, free, T, num_pages=P, free_count=count)
            ops.rope_axes_insert(q, k, v, torch.cat([t.positions[None], axes]), sections, kv, t.slot_mapping, theta,
                                 out_q=oq)
            ops.paged_fog_chunks(oq, kv[:, :, 0], kv[:, :, 1], table, t.query_start_loc, t.seq_lens, fog_alpha=0.0,
                                 out=out)
            return t
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                t = run()
            graph.replay()
            graph.replay()
        else:
            t = run()
        torch.cuda.synchronize()
        row = 0
        for r in range(R):
            have = sum(len(x) for x in hist[r])
            pos = torch.cat([torch.arange(have, have + new[r], device="cuda")[None].int(), axes[:, row:row + new[r]]])
            wq, _ = _rotate64(q[row:row + new[r]], pos.cpu().numpy(), sections, theta, False)
            wk, _ = _rotate64(k[row:row + new[r]], pos.cpu().numpy(), sections, theta, False)
            hist[r].append(torch.cat([torch.from_numpy(wk).cuda(), v[row:row + new[r]].double()], 1))
            if new[r]:
                past = torch.cat(hist[r])
                x = torch.einsum("thd,shd->hts", torch.from_numpy(wq).cuda(),
                                 past[:, :Hkv].repeat_interleave(Hq // Hkv, 1)) / math.sqrt(D)
                at = torch.arange(have, have + new[r], device="cuda")
                x = x.masked_fill(torch.arange(have + new[r], device="cuda")[None] > at[:, None], -math.inf)
                w = torch.softmax(x, -1)
                vals = past[:, Hkv:].repeat_interleave(Hq // Hkv, 1)
                want = torch.einsum("hts,shd->thd", w, vals)
                mass = torch.einsum("hts,shd->thd", w, vals.abs())
                # q, k and the probabilities are rounded to bf16 (relative h each): a score moves by at most
                # 2 h sum |q k| / sqrt(D) <= 2 h |q| |k| / sqrt(D) (|q|, |k| about sqrt(D), up to 1.5 sqrt(D))
                h = _half_eps("bf16")
                tol = h * (want.abs() + mass) + 2 * (2 * h * 2.25 * math.sqrt(D)) * mass
                assert ((out[row:row + new[r]].double() - want).abs() <= tol).all()
            row += new[r]
        assert (out[row:] == 5.0).all() and t.slot_mapping[row:].eq(-1).all()
        count.sub_(t.pages_used)
        ctx = t.seq_lens.clone()
    assert count.item() == P - sum(-(-int(c) // ps) for c in ctx)


def test_attention_impl_mixed_step_is_captured_without_a_host_read():
    """KeSSieAttentionImpl.forward of a mixed step inside a CUDA graph, replayed
    with other lengths (the padded batch's rows behind the last token stay)."""
    from types import SimpleNamespace

    from kessie_b200 import kessie_attention as A
    A.KESSIE_STATE.update(fog_alpha=1.5, fog_start=0.5, prompt_len=10, recall_positions=[], recall_boost=0.0)
    A.KESSIE_STATE.enabled = True
    try:
        c = _Case(41, [1, 60, 7, 0], [900, 300, 77, 0], 8, 2, 128, 16, "fp16", layout="vllm", pad=4)
        inner = SimpleNamespace(num_heads=8, num_kv_heads=2, head_size=128, scale=128 ** -0.5, sliding_window=None)
        impl = A.KeSSieAttentionImpl(_inner_impl=inner)
        cache = torch.stack([c.k, c.v])
        md = SimpleNamespace(num_actual_tokens=72, max_query_len=60, query_start_loc=c.start, seq_lens=c.seq,
                             block_table=c.bt)
        out = torch.full((72, 8 * 128), 2.0, dtype=torch.float16, device="cuda")
        impl.forward(None, c.q, None, None, cache, md, out)           # sets up what a first call sets up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            impl.forward(None, c.q, None, None, cache, md, out)
        c.start.copy_(_i32([0, 5, 6, 68, 68]))
        c.seq.copy_(_i32([800, 250, 70, 0]))
        c.q_lens, c.kv_lens = [5, 1, 62, 0], [800, 250, 70, 0]
        out.fill_(2.0)
        graph.replay()
        torch.cuda.synchronize()
        assert (out[68:] == 2.0).all()

        def bias(s):                                                  # in fp16, as torch's operations round it
            fb = int(s * 0.5)
            j = torch.arange(s, device="cuda", dtype=torch.float64).half()
            t = (j.float() / max(fb, 1)).half()
            d = (1.0 - t.float()).half()
            d = (d.float() * d.float()).half()
            return torch.where(torch.arange(s, device="cuda") < fb, (d.float() * -1.5).half(), 0).double()
        c.check(out.view(72, 8, 128), bias=bias)
    finally:
        A.KESSIE_STATE.update(prompt_len=0)
