"""Workloads for timing the operators of the 4-bit cache: writing it, reading it back, attention over it and the document
scores of its keys.  ``own`` chooses between the framework's calls and the same operators in elementary torch operations.

A cache is a pool of pages of 64 tokens.  Keys and values are held per (token, KV head, 32 channels) as a scale s -- a seventh
of the largest magnitude, rounded to 5 significant bits -- and codes n = round(x / s) in -7..7; the value is n s.

    write   K/V of new tokens go into their slots; read back, so that what is held can be compared
    read    K/V of chosen slots come out of the cache, e.g. documents cached once for a prefill with another query
    attend  query rows (the last tokens of every prompt) over the prompt's pages
    score   the scoring layer's signal rows over the document keys: per-document softmax mass and logits

A prompt is an instruction block, ``docs`` documents of ``doc_lo``..``doc_hi`` tokens (drawn from ``shape_seed``) and a query
block that ends in the tokens generated so far; ``docs`` 0 with ``instr`` 0 is one causal sequence.  ``layout`` is "paged"
(every block begins a page, so that prompts can share the pages of a document) or "packed" (blocks follow one another).
"""
import random

import torch

own = False
PAGE, GROUP = 64, 32
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LARGEST_SCALE = 1.9375 * 2.0 ** 122


def _case(name, kind, prompts, docs, doc_lo, doc_hi, layout="paged", rows=1, ragged=False, lse=False, heads=32, kv_heads=8,
          head_dim=128, dtype="bf16", instr=64, query=48, shape_seed=7):
    return {"name": name, "kind": kind, "prompts": prompts, "docs": docs, "doc_lo": doc_lo, "doc_hi": doc_hi, "layout": layout,
            "rows": rows, "ragged": ragged, "lse": lse, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "instr": instr, "query": query, "shape_seed": shape_seed}


def listed():
    return [
        # one decoding step of a batch: a token of each prompt goes into the cache (rows: new tokens at a prompt's end)
        _case("write_step_32prompts", "write", 32, 5, 35, 90, rows=1),
        # a small model kept in 32 bits caches short ragged prompts
        _case("write_12docs_f32_d64", "write", 2, 12, 17, 120, layout="packed", rows=0, heads=8, kv_heads=2, head_dim=64, dtype="f32"),
        # the benchmark's batch after prefill: every token of 4 prompts of 100 documents, one layer
        _case("write_100docs", "write", 4, 100, 160, 160, rows=0),
        # one document's K/V back for a prefill with another query
        _case("read_1doc", "read", 1, 1, 133, 133),
        # a prompt of 100 documents put together from cached ones, in an order of its own
        _case("read_100docs_ragged", "read", 4, 100, 32, 256),
        # one request, a handful of passages, one answer token: latency
        _case("attend_step_5docs", "attend", 1, 5, 35, 90, instr=27, query=19),
        # a served batch: 16 prompts of 100 documents of different lengths, one answer token each
        _case("attend_step_16prompts", "attend", 16, 100, 32, 256),
        # two long contexts of one causal sequence, one token each
        _case("attend_step_long", "attend", 2, 0, 0, 0, layout="packed", instr=0, query=131071, lse=True),
        # a new query block over cached documents: as many rows as the block has tokens, different in each prompt
        _case("attend_query_block", "attend", 4, 100, 160, 160, rows=48, ragged=True),
        # a small model in 32 bits, three tokens at a time (a drafted answer being verified)
        _case("attend_3rows_f32_d64", "attend", 3, 20, 17, 120, layout="packed", rows=3, ragged=True, heads=8, kv_heads=4,
              head_dim=64, dtype="f32", lse=True),
        # ranking one short request from the cache
        _case("score_5docs", "score", 1, 5, 35, 90, layout="packed", rows=2, instr=27, query=19),
        # ranking a batch of long lists from the cache
        _case("score_16prompts", "score", 16, 100, 32, 256, rows=2),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "score"])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128)] * 3 + [(8, 2, 128), (16, 2, 128), (16, 16, 128), (8, 4, 64), (16, 8, 64), (7, 7, 64)])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    rows = 2 if kind == "score" else _log_int(rng, 1, 48) if rng.random() < 0.4 else 1
    if kind == "write" and rng.random() < 0.5:
        rows = 0
    budget = 60000 if kind in ("write", "read") else 220000 // rows if dtype == "bf16" else 60000 // rows  # slots of one call
    budget = min(budget, budget * 1024 // (kv_heads * head_dim))
    instr, query = rng.randint(1, 130), rng.randint(max(rows, 1), 70)
    if kind == "attend" and rng.random() < 0.25:  # one causal sequence
        prompts = _log_int(rng, 1, 32)
        query = _log_int(rng, rows, max(rows + 1, budget // prompts))
        docs = doc_lo = doc_hi = instr = 0
        layout = "packed"
    else:
        doc_hi = _log_int(rng, 1, 300)
        doc_lo = rng.randint(max(1, doc_hi // 8), doc_hi)
        layout = rng.choice(["paged", "packed"])
        unit = max(doc_hi, PAGE) if layout == "paged" else doc_hi
        docs = _log_int(rng, 1, max(1, min(300, budget // unit)))
        prompts = _log_int(rng, 1, max(1, min(32, budget // (docs * unit + instr + query))))
    c = _case("", kind, prompts, docs, doc_lo, doc_hi, layout, rows, rows > 1 and rng.random() < 0.5,
              kind == "attend" and rng.random() < 0.3, heads, kv_heads, head_dim, dtype, instr, query, rng.randrange(1 << 20))
    del c["name"]
    return c


def _shapes(case):
    """(block lengths, block starts, pages of the longest prompt, query rows), each but the third by prompt."""
    rng = random.Random(case["shape_seed"])
    lens, starts, q_len = [], [], []
    for _ in range(case["prompts"]):
        docs = [rng.randint(case["doc_lo"], case["doc_hi"]) for _ in range(case["docs"])]
        bl = ([case["instr"]] if case["docs"] or case["instr"] else []) + docs + [case["query"] + (1 if case["kind"] == "attend" and case["rows"] == 1 else 0)]
        at, st = 0, []
        for n in bl:
            st.append(at)
            at += n if case["layout"] == "packed" else -(-n // PAGE) * PAGE
        lens.append(bl)
        starts.append(st)
        q_len.append(rng.randint(1, case["rows"]) if case["ragged"] else case["rows"])
    return lens, starts, max(-(-(s[-1] + n[-1]) // PAGE) for n, s in zip(lens, starts)), q_len


def _inputs(case, seed):
    """What both forms start from: spans, page table, K and V of every slot of the pool, queries."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    lens, starts, n_pages, q_len = _shapes(case)
    B, Nk, D = case["prompts"], case["kv_heads"], case["head_dim"]
    start = torch.tensor(starts, dtype=torch.int32, device=dev)
    length = torch.tensor(lens, dtype=torch.int32, device=dev)
    pool = B * n_pages + 3
    table = torch.randperm(pool, generator=gen, device=dev)[:B * n_pages].reshape(B, n_pages).to(torch.int32)

    def states(*shape, spread):
        """Activations whose channels differ in size, as a model's keys do; some tokens far larger than others."""
        x = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)
        channel = torch.exp(spread * torch.randn(shape[-2:], generator=gen, device=dev))
        token = torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=gen, device=dev))
        return (x * channel * token).to(dt)

    t = {"start": start, "length": length, "table": table, "pool": pool, "scale": D ** -0.5,
         "q_len": torch.tensor(q_len, dtype=torch.int32, device=dev)}
    slot = torch.arange(n_pages * PAGE, device=dev)
    inside = ((slot[None, :, None] >= start[:, None]) & (slot[None, :, None] < (start + length)[:, None])).any(-1)
    physical = table.long().repeat_interleave(PAGE, 1) * PAGE + slot % PAGE
    if case["kind"] == "write":
        if case["rows"]:  # the newest tokens of every prompt
            end = (start + length)[:, -1:].long()
            at = end - case["rows"] + torch.arange(case["rows"], device=dev)
            t["slots"] = physical.gather(1, at).to(torch.int32)
        else:  # every token; slots outside the blocks are padding
            t["slots"] = torch.where(inside, physical, -1).to(torch.int32)
        S = t["slots"].shape[1]
        t["k"], t["v"] = (states(B, S, Nk, D, spread=s).transpose(1, 2) for s in (0.5, 0.2))
        return t
    t["pool_k"], t["pool_v"] = (states(pool * PAGE, Nk, D, spread=s) for s in (0.5, 0.2))
    if case["kind"] == "read":  # the prompt's blocks with the documents in another order
        order = torch.argsort(torch.rand(B, n_pages, generator=gen, device=dev), 1)
        pages = lambda x: x.reshape(B, n_pages, PAGE).gather(1, order[..., None].expand(-1, -1, PAGE)).reshape(B, -1)
        t["slots"] = pages(torch.where(inside, physical, -1)).to(torch.int32)
    else:
        t["q"] = states(B, case["rows"], case["heads"], D, spread=0.3).transpose(1, 2)
    return t


# ---- plain form ---------------------------------------------------------------------------------
def _hold(x):
    """(..., D) -> int8 codes (..., D) and fp32 scales (..., D / 32).  The quotients are taken in 64 bits: values lie on borders."""
    g = x.double().unflatten(-1, (-1, GROUP))
    seventh = g.abs().amax(-1) / 7
    quantum = torch.exp2(torch.frexp(seventh).exponent.clamp_min(-125).double() - 5)
    s = (torch.round(seventh / quantum) * quantum).clamp_max(LARGEST_SCALE)
    n = torch.round(g / torch.where(s > 0, s, 1)[..., None]).clamp(-7, 7)
    return n.flatten(-2).to(torch.int8), s.float()


def _values(codes, scales):
    return (codes.unflatten(-1, (-1, GROUP)).float() * scales[..., None]).flatten(-2)


def _pool(codes, scales, t):
    """The values of a prompt's slots, fp32 (B, slots, Nk, D), and whether each lies in a block."""
    slot = torch.arange(t["table"].shape[1] * PAGE, device=t["table"].device)
    at = t["table"].long().repeat_interleave(PAGE, 1) * PAGE + slot % PAGE
    inside = ((slot[None, :, None] >= t["start"][:, None]) & (slot[None, :, None] < (t["start"] + t["length"])[:, None]))
    return _values(codes[at], scales[at]), inside, slot


def _read(t, dtype):
    at, there = t["slots"].long().clamp_min(0), (t["slots"] >= 0)[..., None, None]
    return [torch.where(there, _values(t[n][at], t[n + "_scales"][at]), 0.0).to(dtype).transpose(1, 2) for n in ("codes_k", "codes_v")]


def _write(t):
    there = t["slots"] >= 0
    at = t["slots"][there].long()
    for name, x in (("codes_k", t["k"]), ("codes_v", t["v"])):
        codes, scales = _hold(x.transpose(1, 2)[there])
        t[name][at] = codes
        t[name + "_scales"][at] = scales


def _attend(t):
    k, inside, slot = _pool(t["codes_k"], t["codes_k_scales"], t)
    v = _pool(t["codes_v"], t["codes_v_scales"], t)[0]
    q = t["q"].float()
    B, N, R, D = q.shape
    Nk = k.shape[2]
    row = torch.arange(R, device=q.device)
    row_slot = (t["start"] + t["length"])[:, -1:] - t["q_len"][:, None] + row
    seen = inside.any(-1)[:, None] & (slot <= row_slot[..., None]) & (row < t["q_len"][:, None])[..., None]
    x = torch.matmul(q.reshape(B, Nk, N // Nk * R, D), k.permute(0, 2, 3, 1)).reshape(B, N, R, -1) * t["scale"]
    x = x.masked_fill(~seen[:, None], -float("inf"))
    top = x.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(B, Nk, N // Nk * R, -1), v.transpose(1, 2)).reshape(B, N, R, D)
    out = torch.where(total > 0, out / total, 0.0).to(t["q"].dtype).transpose(1, 2)
    return (out, (top + torch.log(total)).squeeze(-1)) if t["lse"] else out


def _score(t):
    k, inside, _ = _pool(t["codes_k"], t["codes_k_scales"], t)
    docs = inside[..., 1:-1]
    q = t["q"].float()
    B, N, R, D = q.shape
    Nk = k.shape[2]
    x = torch.matmul(q.reshape(B, Nk, N // Nk * R, D), k.permute(0, 2, 3, 1)).reshape(B, N * R, -1) * t["scale"]
    x = x.masked_fill(~docs.any(-1)[:, None], -float("inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    mass = torch.matmul(p, docs.float()) / p.sum(-1, keepdim=True)
    return mass.reshape(B, N, R, -1), mass.mean(1) / t["temperature"]


# ---- the tools' interface -----------------------------------------------------------------------
def prepare(case, seed):
    t = _inputs(case, seed)
    t |= {"kind": case["kind"], "dtype": DTYPES[case["dtype"]], "lse": case["lse"], "temperature": 0.05}
    t["max_block_len"] = max(max(n) for n in _shapes(case)[0])
    Nk, D, pool = case["kv_heads"], case["head_dim"], t["pool"]
    k, v = t.pop("pool_k", None), t.pop("pool_v", None)
    if own:
        from blockrank_b200 import ops
        t["ops"], t["cache"] = ops, ops.cache_alloc(pool, Nk, D, device="cuda")
        if k is not None:
            every = torch.arange(pool * PAGE, dtype=torch.int32, device="cuda")[None]
            ops.cache_write(k[None].transpose(1, 2), v[None].transpose(1, 2), t["cache"], every)
    else:
        for name, x in (("codes_k", k), ("codes_v", v)):
            if x is None:
                t[name] = torch.zeros(pool * PAGE, Nk, D, dtype=torch.int8, device="cuda")
                t[name + "_scales"] = torch.zeros(pool * PAGE, Nk, D // GROUP, device="cuda")
            else:
                t[name], t[name + "_scales"] = _hold(x)
    return t


def run(state):
    t, kind = state, state["kind"]
    if own:
        ops = t["ops"]
        if kind == "attend":
            return ops.cache_attention(t["q"], t["cache"], t["table"], t["start"], t["length"], t["scale"], q_len=t["q_len"],
                                       return_lse=t["lse"])
        if kind == "score":
            return ops.cache_doc_scores(t["q"], t["cache"], t["table"], t["start"], t["length"], t["scale"], t["max_block_len"],
                                        temperature=t["temperature"])
        if kind == "write":
            ops.cache_write(t["k"], t["v"], t["cache"], t["slots"])
        return ops.cache_read(t["cache"], t["slots"], dtype=t["dtype"])
    if kind == "attend":
        return _attend(t)
    if kind == "score":
        return _score(t)
    if kind == "write":
        _write(t)
    return _read(t, t["dtype"])


def work(case):
    lens, _, n_pages, q_len = _shapes(case)
    B, N, Nk, D, e = case["prompts"], case["heads"], case["kv_heads"], case["head_dim"], 2 if case["dtype"] == "bf16" else 4
    held = D // 2 + 2 * D // GROUP  # bytes of a token's key (or value) in one head
    if case["kind"] == "write":
        slots = B * (case["rows"] or n_pages * PAGE)
        tokens = B * case["rows"] if case["rows"] else sum(map(sum, lens))
        # read: the values of the tokens, the slots; write: what is held of them; the read back writes every slot it is given
        return {"bytes": 2 * Nk * (tokens * (e * D + held) + slots * e * D) + 4 * slots, "flops": 2 * Nk * tokens * D * 4}
    if case["kind"] == "read":
        slots, tokens = B * n_pages * PAGE, sum(map(sum, lens))
        return {"bytes": 2 * Nk * (tokens * held + slots * e * D) + 4 * slots, "flops": 2 * Nk * tokens * D}
    if case["kind"] == "score":
        tokens, rows, docs = sum(sum(bl[1:-1]) for bl in lens), B * N * case["rows"], case["docs"]
        return {"bytes": tokens * Nk * held + e * D * rows + 4 * docs * (rows + B) + 4 * B * n_pages, "flops": 2 * D * N * case["rows"] * tokens}
    pairs = sum(r * sum(bl) - r * (r - 1) // 2 for bl, r in zip(lens, q_len))
    rows = B * N * case["rows"]
    return {"bytes": 2 * Nk * held * sum(map(sum, lens)) + 2 * e * D * rows + 4 * B * n_pages + (4 * rows if case["lse"] else 0),
            "flops": 4 * D * N * pairs}


# ---- 64 bits ------------------------------------------------------------------------------------
def _held_exactly(x):
    """The values that the cache holds for x (..., D), in 64 bits: codes by counting the borders below each magnitude."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    a = g.abs()
    target = a.max(-1, keepdim=True).values / 7
    low = torch.full_like(target, 2.0 ** -130)
    step = torch.maximum(torch.exp2(torch.floor(torch.log2(torch.maximum(target, low)))) / 16, low)
    # (log2 may be off by one next to a power of two)
    step = torch.maximum(torch.where(target / step >= 32, step * 2, torch.where(target / step < 16, step / 2, step)), low)
    down = torch.floor(target / step)
    rest = target / step - down
    up = (rest > 0.5) | ((rest == 0.5) & (down % 2 == 1))
    s = ((down + up) * step).clamp_max(LARGEST_SCALE)
    n = torch.zeros_like(a)
    for k in range(1, 8):
        border = (k - 0.5) * s
        n += (a > border) | ((a == border) & (k % 2 == 0))
    return (torch.where(s > 0, n, 0.0) * torch.sign(g) * s).reshape(x.shape)


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "write":
        there = (t["slots"] >= 0)[:, None, :, None]
        return [torch.where(there, _held_exactly(x), 0.0) for x in (t["k"], t["v"])]
    k, v = _held_exactly(t["pool_k"]), _held_exactly(t["pool_v"])
    if case["kind"] == "read":
        there, at = (t["slots"] >= 0)[:, :, None, None], t["slots"].clamp_min(0).long()
        return [torch.where(there, x[at], 0.0).permute(0, 2, 1, 3) for x in (k, v)]
    lens, starts, n_pages, q_len = _shapes(case)
    outs, lses, masses = [], [], []
    G = case["heads"] // case["kv_heads"]
    for b, (bl, st, rows) in enumerate(zip(lens, starts, q_len)):
        slots = [torch.arange(s, s + n, device="cuda") for s, n in zip(st, bl)]
        q = t["q"][b].double()
        if case["kind"] == "score":
            slots = slots[1:-1]
        j = torch.cat(slots)
        at = t["table"][b].long()[j // PAGE] * PAGE + j % PAGE
        x = torch.einsum("hrd,jhd->hrj", q, k[at].repeat_interleave(G, 1)) * t["scale"]
        if case["kind"] == "score":
            p = torch.softmax(x, -1)
            masses.append(torch.stack([c.sum(-1) for c in p.split([len(s) for s in slots], -1)], -1))
            continue
        last = st[-1] + bl[-1] - rows + torch.arange(case["rows"], device="cuda")
        x = x.masked_fill(j[None] > last[:, None], -torch.inf)[:, :rows]
        o = torch.einsum("hrj,jhd->rhd", torch.softmax(x, -1), v[at].repeat_interleave(G, 1))
        pad = case["rows"] - rows
        outs.append(torch.nn.functional.pad(o, (0, 0, 0, 0, 0, pad)))
        lses.append(torch.nn.functional.pad(torch.logsumexp(x, -1), (0, pad), value=-torch.inf))
    if case["kind"] == "score":
        mass = torch.stack(masses)
        return mass, mass.mean((1, 2)) / 0.05
    out = torch.stack(outs)
    return (out, torch.stack(lses)) if case["lse"] else out
