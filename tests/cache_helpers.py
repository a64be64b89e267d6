"""The 4-bit cache in 64 bits, on the CPU: what is held, and attention and document scores over held values."""
import torch

PAGE = 64


def scales(x):
    """(..., D) -> fp64 (..., D/32): max|x| / 7 rounded to 5 significant bits, NaN where the group is not finite."""
    a = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    a = torch.where(x.double().unflatten(-1, (-1, 32)).isfinite().all(-1), a, torch.nan)
    seventh = torch.nan_to_num(a, nan=0.0) / 7
    _, e = torch.frexp(seventh)
    quantum = torch.ldexp(torch.ones_like(seventh), e.clamp_min(-125) - 5)
    s = (torch.round(seventh / quantum) * quantum).clamp_max(1.9375 * 2.0 ** 122)
    return torch.where(a.isnan(), a, s)


def held(x):
    """The values that the cache holds for x, fp64 (torch.round goes to even)."""
    s = scales(x)[..., None]
    g = x.double().unflatten(-1, (-1, 32))
    n = torch.where(s > 0, torch.round(g / torch.where(s > 0, s, 1.0)).clamp(-7, 7), 0.0)
    return (n * s).flatten(-2)


def spans(lens, paged, gap=0):
    """Block lengths per prompt -> start, len int32 (B, M) and the number of page-table entries."""
    start, most = [], 0
    for bl in lens:
        at, st = 0, []
        for n in bl:
            st.append(at)
            at += (-(-n // PAGE) * PAGE if paged else n) + gap
        start.append(st)
        most = max(most, at)
    return torch.tensor(start, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32), -(-max(most, 1) // PAGE)


def slots_of(table, s):
    """Pool slots of the logical slots s of one prompt."""
    return table.long()[s // PAGE] * PAGE + s % PAGE


def visible(start, length, row_slot):
    """Logical slots that a row at row_slot sees (one prompt)."""
    s = torch.cat([torch.arange(a, a + n) for a, n in zip(start.tolist(), length.tolist())])
    return s[s <= row_slot]


def attention(q, k, v, table, start, length, scale, q_len=None):
    """q (B,N,L,D); k, v fp64 held values (pool slots, Nk, D).  Returns out (B,L,N,D), lse (B,N,L) and a bound on what one relative
    unit of error in every product and sum does to a logit (B,N,L): scale * sum |q||k| at most."""
    B, N, R, D = q.shape
    G = N // k.shape[1]
    out = torch.zeros(B, R, N, D, dtype=torch.float64)
    lse = torch.full((B, N, R), -torch.inf, dtype=torch.float64)
    size = torch.zeros(B, N, R, dtype=torch.float64)
    for b in range(B):
        rows = R if q_len is None else int(q_len[b])
        for i in range(rows):
            s = visible(start[b], length[b], int(start[b, -1] + length[b, -1]) - rows + i)
            at = slots_of(table[b], s)
            kk, vv = (x[at].repeat_interleave(G, 1) for x in (k, v))
            x = torch.einsum("hd,jhd->hj", q[b, :, i].double(), kk) * scale
            size[b, :, i] = torch.einsum("hd,jhd->hj", q[b, :, i].double().abs(), kk.abs()).amax(1) * scale
            lse[b, :, i] = torch.logsumexp(x, -1)
            out[b, i] = torch.einsum("hj,jhd->hd", torch.softmax(x, -1), vv)
    return out, lse, size


def doc_mass(q, k, table, start, length, scale):
    B, N, R, D = q.shape
    G, nd = N // k.shape[1], start.shape[1] - 2
    mass = torch.zeros(B, N, R, nd, dtype=torch.float64)
    for b in range(B):
        docs = [torch.arange(int(s), int(s) + int(n)) for s, n in zip(start[b, 1:-1], length[b, 1:-1])]
        if sum(map(len, docs)) == 0:
            continue
        kk = k[slots_of(table[b], torch.cat(docs))].repeat_interleave(G, 1)
        p = torch.softmax(torch.einsum("hrd,jhd->hrj", q[b].double(), kk) * scale, -1)
        mass[b] = torch.stack([c.sum(-1) for c in p.split([len(d) for d in docs], -1)], -1)
    return mass
