"""Cases of the scheduler-step operators: step tables, multi-axis rotary with
slot insert, and attention of ragged chunks over the paged KV cache.

A serving step runs them in this order: the lengths of the running requests
become page tables and slots, the new tokens' q and k are rotated and k, v
written to their slots, and every request's new tokens attend to its cached
keys.  `run` computes one of them, in elementary torch operations (own False)
or through the library (own True).
"""

import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


# ----------------------------------------------------------------- cases
def _chunks(name, dtype, batch, chunks, chunk_lo, chunk_hi, tail_hi, ctx_lo, ctx_hi, hq, hkv, dim, page, window=0,
            fog="none", pad=0, causal=True, lens=1):
    return {"name": name, "op": "chunks", "dtype": dtype, "batch": batch, "chunks": chunks, "chunk_lo": chunk_lo,
            "chunk_hi": chunk_hi, "tail_hi": tail_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "hq": hq, "hkv": hkv,
            "dim": dim, "page": page, "window": window, "fog": fog, "pad": pad, "causal": causal, "lens": lens}


def _insert(name, dtype, tokens, hq, hkv, dim, page, half, axes, interleaved, theta, far, lens=1):
    return {"name": name, "op": "insert", "dtype": dtype, "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim,
            "page": page, "half": half, "axes": axes, "interleaved": interleaved, "theta": theta, "far": far,
            "lens": lens}


def _remap(name, dtype, tokens, heads, dim, half, axes, interleaved, theta, far, lens=1):
    return {"name": name, "op": "remap", "dtype": dtype, "tokens": tokens, "hkv": heads, "dim": dim, "half": half,
            "axes": axes, "interleaved": interleaved, "theta": theta, "far": far, "lens": lens}


def _tables(name, batch, chunks, chunk_lo, chunk_hi, tail_hi, ctx_lo, ctx_hi, page, pad, lens=1):
    return {"name": name, "op": "tables", "batch": batch, "chunks": chunks, "chunk_lo": chunk_lo,
            "chunk_hi": chunk_hi, "tail_hi": tail_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "page": page, "pad": pad,
            "lens": lens}


def listed():
    return [
        # a few short conversations, some answering and some reading a short prompt: the launch counts
        _chunks("chunks_short", "fp16", 6, 3, 5, 64, 1, 30, 600, 8, 2, 64, 16, fog="values", lens=11),
        # a decode step of 28 conversations in a batch padded to 32 rows, as a captured graph runs it
        _chunks("chunks_decode_padded", "bf16", 28, 0, 0, 0, 1, 1000, 16000, 32, 8, 128, 16, pad=4, lens=12),
        # a mixed step: most requests answer, four read their next chunk, the fog on the scores
        _chunks("chunks_mixed", "bf16", 16, 4, 96, 512, 1, 2000, 32768, 32, 8, 128, 32, fog="scores", lens=13),
        # draft tokens being verified, a few per request, under a sliding window
        _chunks("chunks_verify_window", "bf16", 24, 24, 2, 6, 1, 500, 20000, 64, 8, 128, 16, window=4096, lens=14),
        # the rest of one prompt, 17 tokens, behind a 262,127-key context
        _chunks("chunks_long_tail", "fp16", 1, 1, 17, 17, 1, 262110, 262110, 64, 8, 128, 16, fog="values", lens=15),
        # one 4,096-token chunk of a long document
        _chunks("chunks_prefill", "bf16", 1, 1, 4096, 4096, 1, 126976, 126976, 32, 8, 128, 16, fog="values", lens=16),
        # the new tokens of a decode step
        _insert("rope_insert_decode", "bf16", 32, 32, 8, 128, 16, 64, 3, False, 1000000.0, 131072, lens=21),
        # a chunk holding image patches, axes interleaved over the frequencies
        _insert("rope_insert_chunk", "bf16", 8197, 32, 8, 128, 16, 64, 3, True, 5000000.0, 32768, lens=22),
        # fp32 rows, half of the head rotated, two axes
        _insert("rope_insert_fp32", "fp32", 1027, 8, 2, 64, 16, 16, 2, False, 10000.0, 1048576, lens=23),
        # recalled image and text keys moved to new positions
        _remap("rope_remap_recall", "fp16", 65536, 8, 128, 64, 3, False, 1000000.0, 262144, lens=31),
        # eight requests starting a step
        _tables("tables_small", 8, 2, 100, 250, 1, 0, 8000, 16, 0, lens=41),
        # two thousand requests, a hundred of them with long chunks, padded to the captured size
        _tables("tables_large", 2048, 128, 512, 2048, 4, 0, 32768, 16, 1000, lens=42),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["chunks", "chunks", "chunks", "insert", "remap", "tables"])
    seed = rng.randrange(1 << 30)
    if op == "chunks":
        dim = rng.choice([64, 128, 128])
        hkv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 7, 8, 16])
        batch = _log_int(rng, 1, 48)
        chunk_hi = _log_int(rng, 2, 1500)
        ctx_hi = _log_int(rng, 20, 60000)
        case = _chunks("", rng.choice(["bf16", "fp16"]), batch, rng.randint(0, min(batch, 6)), max(1, chunk_hi // 8),
                       chunk_hi, rng.choice([1, 1, 5]), max(1, ctx_hi // 40), ctx_hi, hkv * group, hkv, dim,
                       rng.choice([16, 32, 64]), window=rng.choice([0, 0, 100, 4096]),
                       fog=rng.choice(["none", "values", "scores"]), pad=rng.choice([0, 3]), lens=seed)
        while work(case)["flops"] > 8e12 or work(case)["bytes"] > 1e9:       # no more than the largest listed
            case["ctx_hi"] = case["ctx_hi"] // 2
            case["ctx_lo"] = max(1, case["ctx_hi"] // 40)
            case["chunk_hi"] = max(2, case["chunk_hi"] * 2 // 3)
            case["chunk_lo"] = max(1, case["chunk_hi"] // 8)
    elif op in ("insert", "remap"):
        dim = rng.choice([64, 128])
        half = rng.choice([dim // 2, dim // 2, dim // 4])
        axes = rng.randint(1, 4)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        hkv = rng.choice([1, 2, 4, 8])
        args = (half, axes, rng.random() < 0.5, rng.choice([10000.0, 500000.0, 1000000.0]),
                _log_int(rng, 1000, 1 << 20))
        if op == "insert":
            case = _insert("", dtype, _log_int(rng, 1, 8000), hkv * rng.choice([1, 3, 4, 8]), hkv, dim,
                           rng.choice([16, 32, 64]), *args, lens=seed)
        else:
            case = _remap("", dtype, _log_int(rng, 1, 60000), hkv, dim, *args, lens=seed)
    else:
        batch = _log_int(rng, 1, 2000)
        chunk_hi = _log_int(rng, 2, 2000)
        case = _tables("", batch, rng.randint(0, min(batch, 100)), max(1, chunk_hi // 8), chunk_hi,
                       rng.choice([1, 4]), 0, _log_int(rng, 10, 32768), rng.choice([16, 32, 64]),
                       rng.choice([0, 5, 333]), lens=seed)
    del case["name"]
    return case


def _lengths(case):
    """(query lengths, lengths with the cached context) of the case's requests."""
    rng = random.Random(case["lens"])
    out = []
    for i in range(case["batch"]):
        n = rng.randint(case["chunk_lo"], case["chunk_hi"]) if i < case["chunks"] else rng.randint(1, case["tail_hi"])
        ctx = rng.randint(0, case["ctx_hi"]) if case["ctx_lo"] == 0 else _log_int(rng, case["ctx_lo"], case["ctx_hi"])
        out.append((n, n + ctx))
    rng.shuffle(out)
    return [n for n, _ in out], [s for _, s in out]


def _sections(case):
    """Frequencies per axis: the last axes get a share each, the first the rest."""
    share = case["half"] * (5 if case["interleaved"] else 6) // 16 if case["axes"] < 4 else case["half"] * 3 // 16
    rest = [share] * (case["axes"] - 1)
    return [case["half"] - sum(rest)] + rest


def _axis_of(sections, interleaved):
    n = len(sections)
    if interleaved:
        return [d % n if d < n * sections[d % n] else 0 for d in range(sum(sections))]
    return [a for a, k in enumerate(sections) for _ in range(k)]


# ----------------------------------------------------------------- state
def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _page_table(gen, lens, page, width, extra):
    """Randomly placed pages: (table int32 [B, width], pages in the pool, the pages left over)."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + extra
    perm = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    o = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[o:o + k]
        o += k
    return table, pool, perm[o:].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "chunks":
        dtype = _DTYPES[case["dtype"]]
        q_lens, kv_lens = _lengths(case)
        ps, hkv, dim = case["page"], case["hkv"], case["dim"]
        table, pool, _ = _page_table(gen, kv_lens, ps, max(-(-n // ps) for n in kv_lens), 2)
        kv = _randn(gen, (pool, ps, 2, hkv, dim), dtype)
        total = sum(q_lens) + case["pad"]
        start = [0]
        for n in q_lens:
            start.append(start[-1] + n)
        state.update(q_lens=q_lens, kv_lens=kv_lens, table=table, k=kv[:, :, 0], v=kv[:, :, 1],
                     q=_randn(gen, (total, case["hq"], dim), dtype) * 1.5,
                     out=torch.zeros(total, case["hq"], dim, dtype=dtype, device="cuda"),
                     start=torch.tensor(start, dtype=torch.int32, device="cuda"),
                     seq=torch.tensor(kv_lens, dtype=torch.int32, device="cuda"),
                     # the newest quarter of each conversation is clear of the fog
                     clear=torch.tensor([max(n * 3 // 4, 1) for n in kv_lens], dtype=torch.int32, device="cuda"),
                     bias=None)
        if own and case["fog"] == "scores":
            from kessie_b200 import ops
            state["bias"] = ops.FogBias(1.5, 0.5, (), 0.0, dtype=torch.float32, device="cuda")
    elif case["op"] in ("insert", "remap"):
        dtype = _DTYPES[case["dtype"]]
        t, dim, axes = case["tokens"], case["dim"], case["axes"]
        state["sections"] = _sections(case)

        def positions():
            return torch.randint(0, case["far"], (axes, t), generator=gen, device="cuda", dtype=torch.int32)
        if case["op"] == "insert":
            ps = case["page"]
            pool = -(-t // ps) + 2
            slots = torch.randperm(pool * ps, generator=gen, device="cuda")[:t].contiguous()
            # one fused projection holds q, k and v of a token next to one another
            qkv = _randn(gen, (t, case["hq"] + 2 * case["hkv"], dim), dtype)
            state.update(q=qkv[:, :case["hq"]], k=qkv[:, case["hq"]:case["hq"] + case["hkv"]],
                         v=qkv[:, case["hq"] + case["hkv"]:], positions=positions(), slots=slots,
                         kv=torch.zeros(pool, ps, 2, case["hkv"], dim, dtype=dtype, device="cuda"),
                         out=torch.empty(t, case["hq"], dim, dtype=dtype, device="cuda"))
        else:
            state.update(k=_randn(gen, (t, case["hkv"], dim), dtype), orig=positions(), target=positions(),
                         out=torch.empty(t, case["hkv"], dim, dtype=dtype, device="cuda"))
    else:
        q_lens, kv_lens = _lengths(case)
        ctx = [s - n for n, s in zip(q_lens, kv_lens)]
        ps = case["page"]
        new = sum(-(-s // ps) - -(-c // ps) for c, s in zip(ctx, kv_lens))
        table, pool, free = _page_table(gen, ctx, ps, max(-(-s // ps) for s in kv_lens), new + 7)
        state.update(ctx=torch.tensor(ctx, dtype=torch.int32, device="cuda"),
                     new=torch.tensor(q_lens, dtype=torch.int32, device="cuda"), table=table, free=free,
                     num_tokens=sum(q_lens) + case["pad"], num_pages=pool)
    return state


# ----------------------------------------------------------------- passes
def run(state):
    op = state["case"]["op"]
    if own:
        return {"chunks": _own_chunks, "insert": _own_insert, "remap": _own_remap, "tables": _own_tables}[op](state)
    return {"chunks": _plain_chunks, "insert": _plain_insert, "remap": _plain_remap, "tables": _plain_tables}[op](state)


def _own_chunks(state):
    from kessie_b200 import ops
    case = state["case"]
    fog = case["fog"]
    return ops.paged_fog_chunks(state["q"], state["k"], state["v"], state["table"], state["start"], state["seq"],
                                clear_start=state["clear"] if fog == "values" else None,
                                fog_alpha=0.5 if fog == "values" else 0.0, window_size=case["window"],
                                causal=case["causal"], bias=state["bias"], out=state["out"])


def _own_insert(state):
    from kessie_b200 import ops
    case = state["case"]
    out = ops.rope_axes_insert(state["q"], state["k"], state["v"], state["positions"], state["sections"], state["kv"],
                               state["slots"], rope_theta=case["theta"], interleaved=case["interleaved"],
                               out_q=state["out"])
    return out, state["kv"]


def _own_remap(state):
    from kessie_b200 import ops
    case = state["case"]
    return ops.rope_axes_remap(state["k"], state["orig"], state["target"], state["sections"], rope_theta=case["theta"],
                               interleaved=case["interleaved"], out=state["out"])


def _own_tables(state):
    from kessie_b200 import ops
    t = ops.step_tables(state["ctx"], state["new"], state["table"], state["case"]["page"], state["free"],
                        state["num_tokens"], num_pages=state["num_pages"])
    return t.query_start_loc, t.seq_lens, t.positions, t.slot_mapping, t.pages_used, state["table"]


def _plain_chunks(state):
    case, out = state["case"], state["out"]
    hkv, dim, ps = case["hkv"], case["dim"], case["page"]
    g = case["hq"] // hkv
    scale = 1.0 / math.sqrt(dim)
    row = 0
    for b, (n, s) in enumerate(zip(state["q_lens"], state["kv_lens"])):
        ids = state["table"][b, :-(-s // ps)].long()
        k = state["k"][ids].reshape(-1, hkv, dim)[:s].float()
        v = state["v"][ids].reshape(-1, hkv, dim)[:s].float()
        q = state["q"][row:row + n].float()
        j = torch.arange(s, device="cuda")
        if case["fog"] == "values":
            cs = state["clear"][b]
            w = torch.where(j < cs, (j.float() / (cs - 1).clamp_min(1).float()).sqrt(), 1.0)
            v = v * w[:, None, None]
        bias = None
        if case["fog"] == "scores":
            edge = int(s * 0.5)
            bias = torch.where(j < edge, -1.5 * (1.0 - j.float() / max(edge, 1)).square(), 0.0)
        step = max(1, (1 << 27) // (g * s))
        for t0 in range(0, n, step):
            t1 = min(n, t0 + step)
            p = s - n + torch.arange(t0, t1, device="cuda")
            seen = torch.ones(t1 - t0, s, dtype=torch.bool, device="cuda")
            if case["causal"] or case["window"]:
                seen &= j[None] <= p[:, None]
            if case["window"]:
                seen &= p[:, None] - j[None] < case["window"]
            for h in range(hkv):
                x = (q[t0:t1, h * g:(h + 1) * g] @ k[:, h].T) * scale
                if bias is not None:
                    x += bias
                x.masked_fill_(~seen[:, None], -math.inf)
                x = torch.exp_(x.sub_(x.amax(-1, keepdim=True)))
                y = (x @ v[:, h]) / x.sum(-1, keepdim=True)
                out[row + t0:row + t1, h * g:(h + 1) * g] = y.to(out.dtype)
        row += n
    return out


def _angles(case, sections, positions):
    half = case["half"]
    freq = torch.tensor([case["theta"] ** (-d / half) for d in range(half)], dtype=torch.float64).float().cuda()
    axis = torch.tensor(_axis_of(sections, case["interleaved"]), device="cuda")
    angle = positions[axis].T.double() * freq.double()
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _rotate(x, cos, sin, half):
    x = x.float()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], dim=-1)


def _plain_insert(state):
    case, kv, out = state["case"], state["kv"], state["out"]
    cos, sin = _angles(case, state["sections"], state["positions"])
    out.copy_(_rotate(state["q"], cos, sin, case["half"]))
    page, slot = state["slots"] // case["page"], state["slots"] % case["page"]
    kv[page, slot, 0] = _rotate(state["k"], cos, sin, case["half"]).to(kv.dtype)
    kv[page, slot, 1] = state["v"]
    return out, kv


def _plain_remap(state):
    case = state["case"]
    cos, sin = _angles(case, state["sections"], state["target"] - state["orig"])
    return state["out"].copy_(_rotate(state["k"], cos, sin, case["half"]))


def _plain_tables(state):
    ps, ctx, new, table, free = state["case"]["page"], state["ctx"], state["new"], state["table"], state["free"]
    total = state["num_tokens"]
    start = torch.zeros(ctx.numel() + 1, dtype=torch.int32, device="cuda")
    start[1:] = torch.cumsum(new, 0)
    seq = ctx + new
    owned, need = (ctx + ps - 1) // ps, (seq + ps - 1) // ps
    first = torch.cumsum(need - owned, 0) - (need - owned)
    col = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (col >= owned[:, None]) & (col < need[:, None])
    j = (first[:, None] + col - owned[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[free.numel() - 1 - j], table))
    t = torch.arange(total, device="cuda")
    r = torch.searchsorted(start[1:].contiguous(), t.int(), right=True).clamp_max(ctx.numel() - 1)
    live = t < start[-1]
    pos = torch.where(live, ctx[r] + t - start[r], 0)
    page = table[r, (pos // ps).clamp_max(table.shape[1] - 1)]
    slots = torch.where(live, page.long() * ps + pos % ps, -1)
    return start, seq, pos.int(), slots, (need - owned).sum().int().reshape(1), table


# ----------------------------------------------------------------- work
def work(case):
    if case["op"] == "chunks":
        q_lens, kv_lens = _lengths(case)
        hq, hkv, dim, w = case["hq"], case["hkv"], case["dim"], case["window"]
        pairs = keys = 0
        for n, s in zip(q_lens, kv_lens):
            first = s - n                                        # position of the first new token
            if not case["causal"] and not w:
                pairs, keys = pairs + n * s, keys + s
                continue
            if w:
                pairs += sum(min(first + t + 1, w) for t in range(n))
                keys += s - max(0, first - w + 1)
            else:
                pairs += n * first + n * (n + 1) // 2
                keys += s
        size = _SIZE[case["dtype"]]
        tables = 4 * sum(-(-s // case["page"]) for s in kv_lens) + 8 * len(q_lens)
        return {"bytes": size * dim * (2 * hkv * keys + 2 * hq * sum(q_lens)) + tables, "flops": 4 * dim * hq * pairs}
    if case["op"] == "insert":
        rows = case["hq"] + 2 * case["hkv"]
        t, size = case["tokens"], _SIZE[case["dtype"]]
        return {"bytes": t * (2 * rows * case["dim"] * size + 4 * case["axes"] + 8),
                "flops": 6 * t * (case["hq"] + case["hkv"]) * case["half"]}
    if case["op"] == "remap":
        t, size = case["tokens"], _SIZE[case["dtype"]]
        return {"bytes": t * (2 * case["hkv"] * case["dim"] * size + 8 * case["axes"]),
                "flops": 6 * t * case["hkv"] * case["half"]}
    q_lens, kv_lens = _lengths(case)
    ps = case["page"]
    new = sum(-(-s // ps) - -(-(s - n) // ps) for n, s in zip(q_lens, kv_lens))
    old = sum(1 for n, s in zip(q_lens, kv_lens) if (s - n) % ps)      # partly filled pages the new tokens go on in
    total = sum(q_lens) + case["pad"]
    return {"bytes": 16 * len(q_lens) + 4 + 12 * total + 8 * new + 4 * old + 4, "flops": 0}


# ----------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The outputs from the definitions, in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "tables":
        return None
    if case["op"] == "chunks":
        return _exact_chunks(case, st)
    half, theta, secs = case["half"], case["theta"], st["sections"]
    moved = (st["positions"] if case["op"] == "insert" else st["target"].double() - st["orig"].double()).double()
    turn = torch.zeros(case["tokens"], half, dtype=torch.float64, device="cuda")
    for d in range(half):
        if case["interleaved"]:
            a = d % len(secs)
            a = a if d < secs[a] * len(secs) else 0
        else:
            a, upto = 0, secs[0]
            while d >= upto:
                a += 1
                upto += secs[a]
        f = float(torch.tensor(theta ** (-d / half), dtype=torch.float64).to(torch.float32))
        turn[:, d] = moved[a] * f
    unit = torch.polar(torch.ones_like(turn), turn)[:, None]

    def spin(x):
        x = x.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * unit
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)
    if case["op"] == "remap":
        return spin(st["k"])
    kv = st["kv"].double()
    flat = kv.permute(2, 0, 1, 3, 4).reshape(2, -1, case["hkv"], case["dim"])
    flat[0][st["slots"]] = spin(st["k"])
    flat[1][st["slots"]] = st["v"].double()
    pages = kv.shape[0]
    return spin(st["q"]), flat.reshape(2, pages, case["page"], case["hkv"], case["dim"]).permute(1, 2, 0, 3, 4)


def _exact_chunks(case, st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    per = case["hq"] // case["hkv"]
    base = 0
    for b in range(len(st["q_lens"])):
        n, s = st["q_lens"][b], st["kv_lens"][b]
        where = torch.arange(s, device="cuda")
        rows = st["table"][b].long()[where // case["page"]], where % case["page"]
        fog = torch.ones(s, dtype=torch.float64, device="cuda")
        lift = torch.zeros(s, dtype=torch.float64, device="cuda")
        if case["fog"] == "values":
            cs = int(st["clear"][b])
            fog[:cs] = (where[:cs].double() / max(cs - 1, 1)) ** 0.5
        elif case["fog"] == "scores":
            edge = int(s * 0.5)
            lift[:edge] = -1.5 * (1 - where[:edge].double() / edge) ** 2
        for head in range(case["hq"]):
            keys = st["k"][rows[0], rows[1], head // per].double()
            vals = st["v"][rows[0], rows[1], head // per].double() * fog[:, None]
            block = max(1, (1 << 26) // s)
            for t0 in range(0, n, block):
                m = min(block, n - t0)
                at = s - n + t0 + torch.arange(m, device="cuda")
                gap = at[:, None] - where[None]
                hide = torch.zeros_like(gap, dtype=torch.bool)
                if case["causal"] or case["window"] > 0:
                    hide |= gap < 0
                if case["window"] > 0:
                    hide |= gap >= case["window"]
                logit = st["q"][base + t0:base + t0 + m, head].double() @ keys.T / math.sqrt(case["dim"]) + lift
                prob = torch.softmax(logit.masked_fill(hide, -math.inf), -1)
                out[base + t0:base + t0 + m, head] = prob @ vals
        base += n
    return out
