"""The 4-bit cache on the GPU against the same in 64 bits."""
import pytest
import torch

from tests import cache_helpers as ch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from blockrank_b200 import _lib, ops

BF16, F32 = torch.bfloat16, torch.float32
PAGE = ch.PAGE


def _rand(*shape, seed, dtype, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(*shape[:-2], 1, shape[-1], generator=g))
    return x.to(dtype)


def _filled(pool, Nk, D, seed, dtype=BF16):
    """A pool of which every slot is written; returns the cache and the held values, fp64 (slots, Nk, D)."""
    k, v = (_rand(pool * PAGE, Nk, D, seed=seed + i, dtype=dtype) for i in (0, 1))
    cache = ops.cache_alloc(pool, Nk, D, "cuda")
    every = torch.arange(pool * PAGE, dtype=torch.int32, device="cuda")[None]
    ops.cache_write(k[None].transpose(1, 2).cuda(), v[None].transpose(1, 2).cuda(), cache, every)
    return cache, ch.held(k), ch.held(v)


def _table(B, P, pool, seed):
    return torch.randperm(pool, generator=torch.Generator().manual_seed(seed))[:B * P].reshape(B, P).to(torch.int32)


def _wide(table, width=4000):
    """The same table with room for far more pages: calls are split in other ways, and many rows go to the tcgen05 kernel however short
    their prompts are."""
    wide = torch.full((table.shape[0], width), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    return wide


def _check(out, lse, ref, ref_lse, size, v, steps):
    """Rounding of the output to its type (half a step), and in front of it: a logit is off by its products' and sums' roundings (at
    most 24 accumulations of 2^-23 of sum |q||k|), a probability by twice that, by its exponential (2^-21) and by what its bf16
    pieces leave out (2^-16 for two), the sums by 2^-23 for each of `steps` accumulations."""
    rel = 2 * float(size.max()) * 24 * 2.0 ** -23 + 2.0 ** -21 + (2.0 ** -16 if out.dtype == BF16 else 0.0) + steps * 2.0 ** -23
    err = (out.double().cpu() - ref).abs()
    allowed = ref.abs() * torch.finfo(out.dtype).eps / 2 + 2 * rel * float(v.abs().max())
    assert bool((err <= allowed).all()), (err - allowed).max()
    if lse is not None:
        dead = ref_lse == -torch.inf
        assert torch.equal(lse.cpu() == -torch.inf, dead)
        err = (lse.double().cpu() - ref_lse)[~dead].abs()
        assert bool((err <= rel + ref_lse[~dead].abs() * 2.0 ** -22).all()), err.max()


# ---- writing and reading -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Nk,S", [(1, 1, 1), (2, 3, 5), (3, 8, 37), (2, 7, 700)])
def test_written_values_are_read_back(dtype, D, B, Nk, S):
    pool = -(-B * S // PAGE) + 2
    k, v = (_rand(B, S, Nk, D, seed=S + i, dtype=dtype, spread=2.0) for i in (0, 1))
    slots = torch.randperm(pool * PAGE, generator=torch.Generator().manual_seed(S))[:B * S].reshape(B, S).to(torch.int32)
    slots[:, ::5] = -1
    cache = ops.cache_alloc(pool, Nk, D, "cuda")
    # (views of a fused projection: heads of a wider row)
    kv = torch.cat([k, v], 2).cuda()
    ops.cache_write(kv[:, :, :Nk].transpose(1, 2), kv[:, :, Nk:].transpose(1, 2), cache, slots.cuda())
    for t in (BF16, F32):
        gk, gv = ops.cache_read(cache, slots.cuda(), t)
        assert gk.dtype == t and gk.shape == (B, Nk, S, D)
        for got, x in ((gk, k), (gv, v)):
            ref = torch.where((slots >= 0)[:, None, :, None], ch.held(x).transpose(1, 2), 0.0)
            assert torch.equal(got.double().cpu(), ref)
    ops.check_status()


def test_values_at_the_ends_of_the_range():
    """Zeros, ties of codes and scales, subnormal and huge magnitudes, NaN and infinities."""
    D, Nk = 64, 1
    rows = []
    half = torch.arange(32) * 0.5 - 8  # s = 1 with the 7 below: every tie
    half[0] = 7.0
    rows.append(half.clamp(-7, 7))
    rows.append(torch.zeros(32))
    rows.append(torch.full((32,), -0.0))
    rows += [torch.linspace(-1, 1, 32) * 2.0 ** e for e in (-149, -140, -133, -130, -126, -100, 100, 122, 126)]
    rows.append(torch.full((32,), torch.finfo(F32).max))
    rows.append(torch.cat([torch.tensor([7 * 1.03125]), torch.linspace(-7.2, 7.2, 31)]))  # s between two 5-bit numbers
    for bad in (torch.nan, torch.inf, -torch.inf):
        r = torch.linspace(-1, 1, 32)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows)
    x = torch.cat([x, x.flip(0)], -1).reshape(1, 1, -1, D)  # (B, Nk, S, D): two groups each
    for dtype in (F32, BF16):
        y = x.to(dtype)
        cache = ops.cache_alloc(1, Nk, D, "cuda")
        slots = torch.arange(y.shape[2], dtype=torch.int32)[None]
        ops.cache_write(y.cuda(), (-y).cuda(), cache, slots.cuda())
        gk, gv = ops.cache_read(cache, slots.cuda(), F32)
        for got, src in ((gk, y), (gv, -y)):
            ref = ch.held(src)
            got = got.double().cpu()
            assert torch.equal(got.isnan(), ref.isnan())
            assert torch.equal(got.nan_to_num(nan=0.0), ref.nan_to_num(nan=0.0))


@pytest.mark.parametrize("S", [7, 1025, 2048, 2049, 3000])
def test_of_tokens_with_the_same_slot_the_last_one_is_kept(S):
    Nk, D, pool = 2, 64, 3
    k, v = (_rand(1, S, Nk, D, seed=i, dtype=F32) for i in (0, 1))
    slots = torch.randint(-1, 40, (1, S), generator=torch.Generator().manual_seed(S), dtype=torch.int32)
    cache, hk, hv = _filled(pool, Nk, D, 5)
    ops.cache_write(k.transpose(1, 2).cuda(), v.transpose(1, 2).cuda(), cache, slots.cuda())
    for i, s in enumerate(slots[0].tolist()):
        if s >= 0:
            hk[s], hv[s] = ch.held(k[0, i]), ch.held(v[0, i])
    every = torch.arange(pool * PAGE, dtype=torch.int32, device="cuda")[None]
    gk, gv = ops.cache_read(cache, every, F32)  # what was not named is what it was
    assert torch.equal(gk[0].transpose(0, 1).double().cpu(), hk) and torch.equal(gv[0].transpose(0, 1).double().cpu(), hv)


@pytest.mark.parametrize("S", [9, 1500, 2500])
def test_slots_outside_the_cache_are_left_out_and_reported(S):
    Nk, D, pool = 1, 128, S // PAGE + 1
    k, v = (_rand(1, S, Nk, D, seed=i, dtype=BF16) for i in (0, 1))
    slots = torch.arange(S, dtype=torch.int32)[None].clone()
    slots[0, 3], slots[0, 5] = pool * PAGE, 2 ** 31 - 1
    cache = ops.cache_alloc(pool, Nk, D, "cuda")
    ops.check_status()
    ops.cache_write(k.transpose(1, 2).cuda(), v.transpose(1, 2).cuda(), cache, slots.cuda())
    with pytest.raises(ValueError, match="slot lies outside the cache"):
        ops.check_status()
    gk, _ = ops.cache_read(cache, slots.cuda())
    with pytest.raises(ValueError, match="slot lies outside the cache"):
        ops.check_status()
    ref = ch.held(k).transpose(1, 2)
    ref[:, :, 3] = ref[:, :, 5] = 0
    assert torch.equal(gk.double().cpu(), ref)


# ---- attention -----------------------------------------------------------------------------------
LENS = {
    "one_token": [[1], [1]],
    "one_block": [[130], [64], [1]],
    "docs": [[5, 64, 1, 100, 33, 20], [1, 63, 65, 128, 2, 9]],
    "empty_docs": [[5, 0, 70, 0, 0, 3], [0, 0, 0, 0, 0, 2], [0, 64, 0, 0, 64, 64]],
    "long": [[40, 900, 700, 12], [40, 1, 1300, 31]],
}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,Nk,D", [(8, 2, 128), (6, 2, 64), (4, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize("name", list(LENS))
@pytest.mark.parametrize("paged", [True, False])
def test_one_row(dtype, N, Nk, D, name, paged):
    start, length, P = ch.spans(LENS[name], paged, gap=0 if paged else 3)
    B = len(LENS[name])
    cache, hk, hv = _filled(B * P + 2, Nk, D, 11, dtype)
    table = _table(B, P, B * P + 2, 3)
    q = _rand(B, 1, N, D, seed=2, dtype=dtype).transpose(1, 2)
    out, lse = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), D ** -0.5, return_lse=True)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, D ** -0.5)
    assert out.shape == (B, 1, N, D) and out.dtype == dtype
    _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
    ops.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,Nk,D", [(8, 2, 128), (6, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("rows", [2, 3, 17, 33, 70])
def test_several_rows_of_different_number(dtype, N, Nk, D, rows):
    lens = [[5, 64, 1, 100, rows + 30], [1, 63, 65, 128, rows], [9, 0, 0, 3, rows + 64], [2, 3, 4, 0, 80]]
    q_len = torch.tensor([rows, rows, rows // 2, 0], dtype=torch.int32)
    start, length, P = ch.spans(lens, False)
    cache, hk, hv = _filled(4 * P + 1, Nk, D, 21, dtype)
    table = _table(4, P, 4 * P + 1, 4)
    q = _rand(4, rows, N, D, seed=6, dtype=dtype).transpose(1, 2)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, D ** -0.5, q_len)
    for tab in (table, _wide(table)):
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), D ** -0.5, q_len=q_len.cuda(), return_lse=True)
        _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
        assert not out[3].any() and not out[2, rows // 2:].any()
    ops.check_status()


@pytest.mark.parametrize("tokens,capacity,B", [(3000, 4096, 1), (70000, 70016, 1), (200, 60000, 2), (33000, 33024, 3)])
def test_long_caches_and_tables_far_longer_than_the_prompt(tokens, capacity, B):
    N, Nk, D, P = 4, 1, 64, -(-capacity // PAGE)
    used = -(-tokens // PAGE)
    cache, hk, hv = _filled(B * used, Nk, D, 31)
    table = torch.full((B, P), -1, dtype=torch.int32)  # entries that no block reaches are never looked at
    table[:, :used] = _table(B, used, B * used, 5)
    start, length = torch.zeros(B, 1, dtype=torch.int32), torch.full((B, 1), tokens, dtype=torch.int32)
    length[-1] -= 77
    q = _rand(B, 2, N, D, seed=7, dtype=BF16).transpose(1, 2)
    out, lse = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), D ** -0.5, return_lse=True)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, D ** -0.5)
    _check(out, lse, ref, ref_lse, size, hv, 12 * used)
    ops.check_status()


def test_views_and_a_given_output():
    N, Nk, D, B, R = 4, 2, 64, 2, 3
    start, length, P = ch.spans([[3, 70, 9], [64, 1, 5]], True)
    cache, hk, hv = _filled(B * P, Nk, D, 41)
    table = _table(B, P, B * P, 6)
    wide = _rand(B, R, N + 2, D, seed=8, dtype=BF16)
    q = wide[:, :, 1:N + 1].transpose(1, 2)
    room = torch.full((B, R + 2, N, D + 16), 7.0, dtype=BF16, device="cuda")
    out = room[:, 1:R + 1, :, :D]
    # page table and spans as columns of something wider
    tab = torch.stack([table, table], -1).cuda()[..., 0]
    st, ln = (torch.stack([x, x], -1).cuda()[..., 0] for x in (start, length))
    got = ops.cache_attention(wide.cuda()[:, :, 1:N + 1].transpose(1, 2), cache, tab, st, ln, 0.2, out=out)
    assert got.data_ptr() == out.data_ptr()
    ref, _, size = ch.attention(q, hk, hv, table, start, length, 0.2)
    _check(out, None, ref, None, size, hv, 3 * P + 8)
    assert (room[:, 0] == 7).all() and (room[:, -1] == 7).all() and (room[..., D:] == 7).all()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype,N,R", [(BF16, 4, 5), (F32, 4, 5), (BF16, 4, 3), (BF16, 16, 5), (BF16, 4, 30)])
def test_what_no_row_sees_has_no_influence(dtype, N, R, wide):
    """Pages of NaN scales and arbitrary codes outside the blocks; NaN and infinities in tokens behind a row's own."""
    Nk, D, B = 2, 128, 2
    lens = [[3, 70, 9, R + 7], [64, 1, 0, R]]
    start, length, P = ch.spans(lens, True, gap=PAGE)
    cache, hk, hv = _filled(B * P + 1, Nk, D, 51, dtype)
    table = _table(B, P, B * P + 1, 7)
    inside = torch.zeros(B * P * PAGE + PAGE, dtype=torch.bool)
    for b in range(B):
        for s, n in zip(start[b].tolist(), length[b].tolist()):
            inside[ch.slots_of(table[b], torch.arange(s, s + n))] = True
    kept_k, kept_v = (x.clone() for x in ops.cache_read(cache, inside.nonzero().T.int().cuda(), F32))
    cache.fill_(255)
    ops.cache_write(kept_k, kept_v, cache, inside.nonzero().T.int().contiguous().cuda())  # (held values are held as they are)
    q = _rand(B, R, N, D, seed=9, dtype=dtype).transpose(1, 2)
    args = (q.cuda(), cache, (_wide(table) if wide else table).cuda(), start.cuda(), length.cuda(), D ** -0.5)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, D ** -0.5)
    out, lse = ops.cache_attention(*args, return_lse=True)
    _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
    # the last token but one of each prompt: NaN in one group of V's first head, an infinity in K's second
    last = (start[:, -1] + length[:, -1] - 2).tolist()
    at = torch.tensor([[int(ch.slots_of(table[b], torch.tensor(last[b])))] for b in range(B)], dtype=torch.int32).cuda()
    k1, v1 = ops.cache_read(cache, at, F32)
    v1[:, 0, 0, 40] = torch.nan
    k1[:, 1, 0, 3] = torch.inf
    ops.cache_write(k1, v1, cache, at)
    bad, bad_lse = ops.cache_attention(*args, return_lse=True)
    assert torch.equal(bad[:, :R - 2], out[:, :R - 2]) and torch.equal(bad_lse[:, :, :R - 2], lse[:, :, :R - 2])
    g = N // Nk
    assert bad[:, R - 2:, :g, 32:64].isnan().all() and bad[:, R - 2:, g:].isnan().all() and bad_lse[:, g:, R - 2:].isnan().all()
    assert torch.equal(bad[:, R - 2:, :g, :32], out[:, R - 2:, :g, :32]) and torch.equal(bad[:, R - 2:, :g, 64:], out[:, R - 2:, :g, 64:])


def test_malformed_prompts_are_left_out_and_reported():
    N, Nk, D, B = 4, 2, 64, 6
    start, length, P = ch.spans([[3, 70, 9]] * B, True)
    cache, hk, hv = _filled(B * P, Nk, D, 61)
    table = _table(B, P, B * P, 8)
    start[1, 1] = 2              # overlaps the first block
    length[2, 2] = P * PAGE      # past the page table
    length[3, 0] = -1
    q_len = torch.tensor([2, 2, 2, 2, 10, 2], dtype=torch.int32)  # prompt 4: more rows than q has and than the last block's 9
    table[5, 0] = B * P          # a page outside the cache: left out, the rest of the prompt is seen
    q = _rand(B, 3, N, D, seed=10, dtype=BF16).transpose(1, 2)
    ops.check_status()
    out = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.3, q_len=q_len.cuda())
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    assert not out[1:5].any()
    for b in (0, 5):
        ln = length[b:b + 1].clone()
        if b == 5:
            ln[0, 0] = 0
        ref, _, size = ch.attention(q[b:b + 1], hk, hv, table[b:b + 1], start[b:b + 1], ln, 0.3, q_len[b:b + 1])
        _check(out[b:b + 1], None, ref, None, size, hv, 32)


def test_pages_beyond_the_reach_of_32_bits():
    """The last pages of a pool of more than 2^32 bytes."""
    N, Nk, D = 8, 8, 128
    pool = 2 ** 32 // 73728 + 40
    cache = ops.cache_alloc(pool, Nk, D, "cuda")
    assert cache.numel() > 2 ** 32
    P, T = 3, 150
    table = torch.tensor([[pool - 1, 5, pool - 2]], dtype=torch.int32)
    k, v = (_rand(1, T, Nk, D, seed=i, dtype=BF16) for i in (1, 2))
    slots = ch.slots_of(table[0], torch.arange(T))[None].int()
    ops.cache_write(k.transpose(1, 2).cuda(), v.transpose(1, 2).cuda(), cache, slots.cuda())
    gk, gv = ops.cache_read(cache, slots.cuda(), F32)
    assert torch.equal(gk.double().cpu(), ch.held(k).transpose(1, 2)) and torch.equal(gv.double().cpu(), ch.held(v).transpose(1, 2))
    q = _rand(1, 1, N, D, seed=3, dtype=BF16).transpose(1, 2)
    start, length = torch.zeros(1, 1, dtype=torch.int32), torch.full((1, 1), T, dtype=torch.int32)
    out = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.1)
    local = torch.arange(P, dtype=torch.int32)[None]
    pad = lambda x: torch.cat([ch.held(x)[0], torch.zeros(P * PAGE - T, Nk, D, dtype=torch.float64)])
    ref, _, size = ch.attention(q, pad(k), pad(v), local, start, length, 0.1)
    _check(out, None, ref, None, size, ch.held(v), 32)
    ops.check_status()


# ---- document scores -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,Nk,D,R", [(8, 2, 128, 2), (6, 2, 64, 1), (4, 4, 64, 2), (16, 2, 128, 3)])
@pytest.mark.parametrize("name", ["docs", "empty_docs", "long"])
@pytest.mark.parametrize("paged", [True, False])
def test_document_scores(dtype, N, Nk, D, R, name, paged):
    start, length, P = ch.spans(LENS[name], paged, gap=0 if paged else 3)
    B = len(LENS[name])
    cache, hk, _ = _filled(B * P + 2, Nk, D, 71, dtype)
    table = _table(B, P, B * P + 2, 9)
    q = _rand(B, R, N, D, seed=12, dtype=dtype).transpose(1, 2)
    mass, logits = ops.cache_doc_scores(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), D ** -0.5, int(length.max()))
    ref = ch.doc_mass(q, hk, table, start, length, D ** -0.5)
    # a probability is off by twice its logit's error (24 accumulations of 2^-23 of sum |q||k|), its exponentials' and the sums'
    size = float((q.double().abs().amax() * hk.abs().sum(-1).amax()) * D ** -0.5)
    rel = 2 * size * 24 * 2.0 ** -23 + 64 * 2.0 ** -23
    assert bool(((mass.double().cpu() - ref).abs() <= rel * ref + 2.0 ** -40).all())
    want = ref.mean((1, 2)) / 0.05
    assert bool(((logits.double().cpu() - want).abs() <= 2 * rel * want + 2.0 ** -40).all())
    ops.check_status()


@pytest.mark.parametrize("paged", [True, False])
def test_scores_of_very_many_documents(paged):
    """More than a CTA looks at in one go, most of them short, some empty, one long."""
    N, Nk, D, R = 4, 2, 64, 2
    g = torch.Generator().manual_seed(3)
    lens = [torch.randint(0, 12, (330,), generator=g).tolist() for _ in range(2)]
    lens[0][17], lens[1][300], lens[1][301] = 900, 2000, 0
    lens = [[7] + x + [5] for x in lens]
    start, length, P = ch.spans(lens, paged)
    cache, hk, _ = _filled(2 * P, Nk, D, 151)
    table = _table(2, P, 2 * P, 17)
    q = _rand(2, R, N, D, seed=18, dtype=BF16).transpose(1, 2)
    mass, logits = ops.cache_doc_scores(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.1, 2000)
    ref = ch.doc_mass(q, hk, table, start, length, 0.1)
    assert torch.allclose(mass.double().cpu(), ref, rtol=1e-4, atol=1e-9)
    assert torch.allclose(logits.double().cpu(), ref.mean((1, 2)) / 0.05, rtol=1e-4, atol=1e-8)
    ops.check_status()


def test_document_scores_are_those_of_the_values_read_back():
    """The cached epilogue against the uncached one on the same numbers."""
    N, Nk, D, R = 32, 8, 128, 2
    lens = [[27, 40, 90, 64, 1, 77, 19], [27, 35, 35, 128, 64, 2, 30]]
    start, length, P = ch.spans(lens, False)
    cache, _, _ = _filled(2 * P, Nk, D, 81)
    table = _table(2, P, 2 * P, 10)
    slots = torch.stack([ch.slots_of(table[b], torch.arange(P * PAGE)) for b in range(2)]).int().cuda()
    k, _ = ops.cache_read(cache, slots)
    rows = torch.tensor([[P * PAGE - 2, P * PAGE - 1]] * 2, dtype=torch.int32).cuda()
    q = _rand(2, P * PAGE, N, D, seed=13, dtype=BF16).transpose(1, 2).cuda()
    want, want_logits = ops.doc_scores(q, k, start.cuda(), length.cuda(), rows, D ** -0.5)
    got, got_logits = ops.cache_doc_scores(q[:, :, -2:], cache, table.cuda(), start.cuda(), length.cuda(), D ** -0.5, int(length.max()))
    assert torch.allclose(got, want, rtol=2e-5, atol=1e-9) and torch.allclose(got_logits, want_logits, rtol=2e-5)


def test_malformed_documents_are_left_out_and_reported():
    N, Nk, D = 4, 2, 64
    start, length, P = ch.spans([[3, 70, 60, 9]] * 3, True)
    cache, hk, _ = _filled(3 * P, Nk, D, 91)
    table = _table(3, P, 3 * P, 11)
    q = _rand(3, 1, N, D, seed=14, dtype=BF16).transpose(1, 2)
    ops.check_status()
    length[1, 1] = 200            # runs into the next block, longer than max_block_len
    table[2, start[2, 1] // PAGE] = -3
    mass, _ = ops.cache_doc_scores(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.2, 70)
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    ref = ch.doc_mass(q[:1], hk, table[:1], start[:1], length[:1], 0.2)
    assert torch.allclose(mass[:1].double().cpu(), ref, rtol=1e-4)
    assert not mass[1, :, :, 0].any()


# ---- together ------------------------------------------------------------------------------------
def test_a_prompt_is_cached_ranked_and_answered():
    """Prefill, the cache filled from its keys and values, document scores, and three decoding steps; two prompts share the pages
    of the instruction and of one document."""
    N, Nk, D = 8, 2, 128
    lens = [[30, 64, 100, 40], [30, 64, 7, 25]]
    start, length, P = ch.spans(lens, True)
    B, S = 2, P * PAGE
    q, k, v = (_rand(B, S, n, D, seed=i, dtype=BF16) for i, n in ((1, N), (2, Nk), (3, Nk)))
    k[1, :128], v[1, :128] = k[0, :128], v[0, :128]  # the same instruction and first document
    table = torch.arange(2 * P, dtype=torch.int32).reshape(2, P).clone()
    table[1, :2] = table[0, :2]
    scale = D ** -0.5
    logical = torch.arange(S)
    inside = [torch.isin(logical, torch.cat([torch.arange(a, a + n) for a, n in zip(start[b].tolist(), length[b].tolist())])) for b in range(B)]
    slots = torch.stack([torch.where(inside[b], ch.slots_of(table[b], logical), -1) for b in range(B)]).int()
    cache = ops.cache_alloc(2 * P, Nk, D, "cuda")
    ops.cache_write(k.cuda().transpose(1, 2), v.cuda().transpose(1, 2), cache, slots.cuda())
    ck, cv = ops.cache_read(cache, slots.cuda())
    st, ln, tab = start.cuda(), length.cuda(), table.cuda()
    # the query block's rows: the prefill attention on what was read back and the cached one agree
    full = ops.attention(q.cuda().transpose(1, 2), ck, cv, st, ln, scale, int(length.max()))
    rows = int(length[:, -1].max())
    qq = torch.zeros(B, rows, N, D, dtype=BF16)
    for b in range(B):
        a, n = int(start[b, -1]), int(length[b, -1])
        qq[b, :n] = q[b, a:a + n]
    got = ops.cache_attention(qq.cuda().transpose(1, 2), cache, tab, st, ln, scale, q_len=ln[:, -1].contiguous())
    for b in range(B):
        a, n = int(start[b, -1]), int(length[b, -1])
        d = (got[b, :n].float() - full[b, a:a + n].float()).abs().max()
        assert d <= 2 ** -7 * float(cv.abs().max())
    mass, logits = ops.cache_doc_scores(qq.cuda().transpose(1, 2)[:, :, :2], cache, tab, st, ln, scale, int(length.max()))
    assert torch.allclose(mass.sum(-1), torch.ones_like(mass.sum(-1)), atol=1e-5) and logits.shape == (B, 2)
    hk, hv = (torch.zeros(2 * P * PAGE, Nk, D, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        hk[slots[b][inside[b]].long()], hv[slots[b][inside[b]].long()] = ch.held(k[b][inside[b]]), ch.held(v[b][inside[b]])
    for step in range(3):
        length[:, -1] += 1
        ln = length.cuda()
        q1, k1, v1 = (_rand(B, 1, n, D, seed=20 + step + i, dtype=BF16) for i, n in ((1, N), (2, Nk), (3, Nk)))
        at = torch.stack([ch.slots_of(table[b], start[b, -1:].long() + length[b, -1:].long() - 1) for b in range(B)]).int()
        ops.cache_write(k1.cuda().transpose(1, 2), v1.cuda().transpose(1, 2), cache, at.cuda())
        hk[at[:, 0].long()], hv[at[:, 0].long()] = ch.held(k1[:, 0]), ch.held(v1[:, 0])
        out = ops.cache_attention(q1.cuda().transpose(1, 2), cache, tab, st, ln, scale)
        ref, _, size = ch.attention(q1.transpose(1, 2), hk, hv, table, start, length, scale)
        _check(out, None, ref, None, size, hv, 32)
    ops.check_status()


def test_a_captured_step_replays_on_new_inputs():
    N, Nk, D, B = 8, 2, 128, 2
    start, length, P = ch.spans([[30, 64, 500, 40], [30, 64, 7, 25]], True)
    cache, hk, hv = _filled(B * P, Nk, D, 101)
    table = _table(B, P, B * P, 12)
    st, ln, tab = start.cuda(), length.cuda(), table.cuda()
    k1, v1, q1 = (torch.zeros(B, 1, n, D, dtype=BF16, device="cuda").transpose(1, 2) for n in (Nk, Nk, N))
    at = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    ops.status_word("cuda")

    def step():
        ops.cache_write(k1, v1, cache, at)
        return ops.cache_attention(q1, cache, tab, st, ln, 0.1), ops.cache_doc_scores(q1, cache, tab, st, ln, 0.1, 512)[0]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        at.fill_(-1)
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same step
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        length[:, -1] += 1
        ln.copy_(length)
        new = [_rand(B, 1, n, D, seed=30 + 3 * i + j, dtype=BF16) for j, n in enumerate((Nk, Nk, N))]
        for dst, src in zip((k1, v1, q1), new):
            dst.copy_(src.transpose(1, 2))
        slot = torch.stack([ch.slots_of(table[b], start[b, -1:].long() + length[b, -1:].long() - 1) for b in range(B)])
        at.copy_(slot)
        hk[slot[:, 0]], hv[slot[:, 0]] = ch.held(new[0][:, 0]), ch.held(new[1][:, 0])
        graph, (out, mass) = graphs[i % 2]
        graph.replay()
        ref, _, size = ch.attention(new[2].transpose(1, 2), hk, hv, table, start, length, 0.1)
        _check(out, None, ref, None, size, hv, 64)
        assert torch.allclose(mass.double().cpu(), ch.doc_mass(new[2].transpose(1, 2), hk, table, start, length, 0.1), rtol=1e-3, atol=1e-6)
    ops.check_status()


def test_calls_on_two_streams_at_once():
    N, Nk, D, B = 8, 2, 128, 2
    start, length, P = ch.spans([[30, 900, 40], [30, 64, 25]], True)
    cache, hk, hv = _filled(B * P, Nk, D, 111)
    table = _table(B, P, B * P, 13)
    qs = [_rand(B, 1, N, D, seed=40 + i, dtype=BF16).transpose(1, 2) for i in range(2)]
    dev = [q.cuda() for q in qs]
    st, ln, tab = start.cuda(), length.cuda(), table.cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ops.cache_attention(dev[i], cache, tab, st, ln, 0.1))
    torch.cuda.synchronize()
    for i in range(2):
        ref, _, size = ch.attention(qs[i], hk, hv, table, start, length, 0.1)
        for out in outs[i]:
            assert torch.equal(out, outs[i][0])
        _check(outs[i][0], None, ref, None, size, hv, 64)


def test_calls_of_nothing():
    cache, _, _ = _filled(2, 2, 64, 121)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    e = lambda *s: torch.zeros(*s, dtype=BF16, device="cuda")
    before = cache.clone()
    ops.cache_write(e(2, 2, 0, 64), e(2, 2, 0, 64), cache, z(2, 0))
    ops.cache_write(e(0, 2, 3, 64), e(0, 2, 3, 64), cache, z(0, 3))
    assert torch.equal(cache, before)
    assert ops.cache_read(cache, z(3, 0))[0].shape == (3, 2, 0, 64)
    assert ops.cache_attention(e(2, 4, 0, 64), cache, z(2, 1), z(2, 1), z(2, 1), 1.0).shape == (2, 0, 4, 64)
    assert ops.cache_attention(e(0, 4, 1, 64), cache, z(0, 1), z(0, 1), z(0, 1), 1.0).shape == (0, 1, 4, 64)
    out, lse = ops.cache_attention(e(2, 4, 3, 64), cache, z(2, 1), z(2, 1), z(2, 1), 1.0, q_len=z(2), return_lse=True)
    assert not out.any() and (lse == -torch.inf).all()
    ops.check_status()


def test_refused_calls():
    cache = ops.cache_alloc(2, 2, 64, "cuda")
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    e = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device="cuda")
    bad = [
        lambda: ops.cache_alloc(0, 2, 64, "cuda"),
        lambda: ops.cache_alloc(2, 2, 96, "cuda"),
        lambda: ops.cache_write(e(1, 2, 3, 64), e(1, 2, 3, 64), cache, z(1, 2)),
        lambda: ops.cache_write(e(1, 2, 3, 64), e(1, 2, 3, 64), cache, z(1, 3).long()),
        lambda: ops.cache_write(e(1, 3, 3, 64), e(1, 3, 3, 64), cache, z(1, 3)),
        lambda: ops.cache_write(e(1, 2, 3, 128), e(1, 2, 3, 128), cache, z(1, 3)),
        lambda: ops.cache_write(e(1, 2, 3, 64), e(1, 2, 3, 64, dtype=F32), cache, z(1, 3)),
        lambda: ops.cache_write(e(1, 2, 3, 64, dtype=torch.float16), e(1, 2, 3, 64, dtype=torch.float16), cache, z(1, 3)),
        lambda: ops.cache_write(e(1, 2, 3, 65)[..., 1:], e(1, 2, 3, 64), cache, z(1, 3)),
        lambda: ops.cache_read(cache, z(3)),
        lambda: ops.cache_read(cache, z(1, 3), torch.float16),
        lambda: ops.cache_read(cache.view(2, 2, 72, 64), z(1, 3)),
        lambda: ops.cache_read(cache[:, :1], z(1, 3)),
        lambda: ops.cache_attention(e(1, 3, 1, 64), cache, z(1, 1), z(1, 1), z(1, 1), 1.0),
        lambda: ops.cache_attention(e(1, 4, 1, 64), cache, z(2, 1), z(1, 1), z(1, 1), 1.0),
        lambda: ops.cache_attention(e(1, 4, 1, 64), cache, z(1, 1), z(1, 1), z(1, 2), 1.0),
        lambda: ops.cache_attention(e(1, 4, 1, 64), cache, z(1, 0), z(1, 1), z(1, 1), 1.0),
        lambda: ops.cache_attention(e(1, 4, 1, 64), cache, z(1, 1), z(1, 1), z(1, 1), 0.0),
        lambda: ops.cache_attention(e(1, 4, 1, 64), cache, z(1, 1), z(1, 1), z(1, 1), float("nan")),
        lambda: ops.cache_attention(e(1, 4, 1, 64), cache, z(1, 1), z(1, 1), z(1, 1), 1.0, q_len=z(2)),
        lambda: ops.cache_attention(e(1, 4, 1, 64), cache, z(1, 1), z(1, 1), z(1, 1), 1.0, out=e(1, 4, 1, 64)),
        lambda: ops.cache_doc_scores(e(1, 4, 1, 64), cache, z(1, 1), z(1, 2), z(1, 2), 1.0, 64),
        lambda: ops.cache_doc_scores(e(1, 4, 1, 64), cache, z(1, 1), z(1, 3), z(1, 3), 1.0, 0),
        lambda: ops.cache_doc_scores(e(1, 4, 65, 64), cache, z(1, 1), z(1, 3), z(1, 3), 1.0, 64),
        lambda: ops.cache_doc_scores(e(1, 4, 1, 64), cache, z(1, 1), z(1, 3), z(1, 3), 1.0, 64, temperature=0.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.cache_read(cache, torch.zeros(1, 3, dtype=torch.int32))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("N,Nk,D,rows,tokens", [(8, 2, 128, 70, 700), (16, 2, 64, 33, 5000), (4, 1, 128, 9, 9000), (8, 1, 64, 100, 131)])
def test_many_rows_over_shares_of_the_pages(N, Nk, D, rows, tokens, wide):
    """Query blocks long enough for the tensor cores' rows, over as many pages as several CTAs take: the same every time."""
    lens = [[40, tokens // 3, tokens // 2, rows], [3, tokens // 4, 64, rows + 7]]
    start, length, P = ch.spans(lens, False)
    cache, hk, hv = _filled(2 * P + 1, Nk, D, 131)
    table = _table(2, P, 2 * P + 1, 14)
    q_len = torch.tensor([rows, rows - 5], dtype=torch.int32)
    q = 3 * _rand(2, rows, N, D, seed=15, dtype=BF16).transpose(1, 2)
    args = (q.cuda(), cache, (_wide(table, 600) if wide else table).cuda(), start.cuda(), length.cuda(), D ** -0.5)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, D ** -0.5, q_len)
    first = None
    for _ in range(30):
        out, lse = ops.cache_attention(*args, q_len=q_len.cuda(), return_lse=True)
        first = first if first is not None else (out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    _check(*first, ref, ref_lse, size, hv, 3 * P + 8)
    ops.check_status()


def test_logits_that_keep_growing():
    """Later pages outweigh earlier ones by far more than a probability can hold: what was summed is brought in line."""
    N, Nk, D, P = 8, 1, 128, 9
    cache, hk, hv = _filled(P, Nk, D, 141)
    k, v = ops.cache_read(cache, torch.arange(P * PAGE, dtype=torch.int32, device="cuda")[None], F32)
    k *= torch.exp2(torch.arange(P * PAGE, device="cuda") / 64.0)[:, None]
    ops.cache_write(k, v, cache, torch.arange(P * PAGE, dtype=torch.int32, device="cuda")[None])
    hk = ch.held(k[0].transpose(0, 1).cpu())
    table = torch.arange(P, dtype=torch.int32)[None]
    start, length = torch.zeros(1, 1, dtype=torch.int32), torch.full((1, 1), P * PAGE - 3, dtype=torch.int32)
    for rows, tab in ((1, table), (2, table), (9, table), (9, _wide(table))):
        q = _rand(1, rows, N, D, seed=16, dtype=BF16).transpose(1, 2)
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), 0.05, return_lse=True)
        ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, 0.05)
        _check(out, lse, ref, ref_lse, size, hv, 64)


@pytest.mark.parametrize("dtype,N,Nk,D,rows", [(BF16, 8, 2, 128, 130), (BF16, 20, 1, 64, 33), (F32, 8, 2, 64, 40), (BF16, 64, 1, 128, 1)])
def test_more_rows_than_a_cta_takes(dtype, N, Nk, D, rows):
    """Several CTAs' rows, their borders inside a token's heads; a prompt without rows, one with fewer than the others."""
    lens = [[40, 130, 0, 61, rows + 2], [3, 5, 64, 1, rows], [1, 700, 2, 2, rows]]
    start, length, P = ch.spans(lens, True)
    cache, hk, hv = _filled(3 * P, Nk, D, 161, dtype)
    table = _table(3, P, 3 * P, 18)
    q_len = torch.tensor([rows, 0, max(1, rows - 9)], dtype=torch.int32)
    q = _rand(3, rows, N, D, seed=19, dtype=dtype).transpose(1, 2)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, D ** -0.5, q_len)
    for tab in (table, _wide(table, 300), _wide(table)):
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), D ** -0.5, q_len=q_len.cuda(), return_lse=True)
        _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
    ops.check_status()


@pytest.mark.parametrize("dtype,rows", [(BF16, 1), (BF16, 9), (BF16, 20), (F32, 3)])
def test_more_blocks_than_a_cta_has_threads(dtype, rows):
    N, Nk, D = 4, 2, 64
    g = torch.Generator().manual_seed(4)
    lens = [[9] + torch.randint(0, 20, (498,), generator=g).tolist() + [rows] for _ in range(2)]
    start, length, P = ch.spans(lens, False, gap=1)
    cache, hk, hv = _filled(2 * P, Nk, D, 171, dtype)
    table = _table(2, P, 2 * P, 20)
    q = _rand(2, rows, N, D, seed=21, dtype=dtype).transpose(1, 2)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, 0.1)
    for tab in (table, _wide(table)):
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), 0.1, return_lse=True)
        _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
    ops.check_status()


def test_a_long_list_of_short_prompts():
    N, Nk, D, B = 4, 2, 64, 600
    lens = [[1 + b % 70] for b in range(B)]
    start, length, P = ch.spans(lens, False)
    cache, hk, hv = _filled(200, Nk, D, 181)
    table = torch.randint(0, 200, (B, P), generator=torch.Generator().manual_seed(5), dtype=torch.int32)  # (prompts share pages)
    q = _rand(B, 1, N, D, seed=22, dtype=BF16).transpose(1, 2)
    out, lse = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.1, return_lse=True)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, 0.1)
    _check(out, lse, ref, ref_lse, size, hv, 64)


@pytest.mark.parametrize("dtype,rows,width", [(BF16, 2, 1), (BF16, 40, 1), (BF16, 2, 4000), (BF16, 40, 4000), (F32, 2, 1), (F32, 40, 4000)])
def test_rows_that_see_nothing(dtype, rows, width):
    """No page of the prompt exists: zeros and -inf, no NaN; the prompts next to it are whole.  Wide tables: parts joined by a kernel."""
    N, Nk, D, B = 4, 2, 64, 4
    start, length, P = ch.spans([[3, 70, rows]] * B, True)
    cache, hk, hv = _filled(B * P, Nk, D, 191, dtype)
    table = torch.full((B, max(P, width)), -1, dtype=torch.int32)
    table[:, :P] = _table(B, P, B * P, 23)
    table[1, :P] = -7
    table[2, :P] = B * P + 5
    q = _rand(B, rows, N, D, seed=24, dtype=dtype).transpose(1, 2)
    ops.check_status()
    out, lse = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.1, return_lse=True)
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    mass, logits = ops.cache_doc_scores(q[:, :, :2].cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.1, 70)
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    assert not out[1:3].any() and (lse[1:3] == -torch.inf).all() and not mass[1:3].any() and not logits[1:3].any()
    length[1:3] = 0
    start[1:3] = 0
    q_len = torch.tensor([rows, 0, 0, rows], dtype=torch.int32)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, 0.1, q_len)
    _check(out, lse, ref, ref_lse, size, hv, 64)
    want = ch.doc_mass(q[:, :, :2], hk, table, start, length, 0.1)
    assert torch.allclose(mass.double().cpu(), want, rtol=1e-4)


@pytest.mark.parametrize("width", [1, 4000])
def test_malformed_prompts_of_many_rows(width):
    N, Nk, D, B, rows = 4, 2, 64, 5, 40
    start, length, P = ch.spans([[3, 70, rows + 2]] * B, True)
    cache, hk, hv = _filled(B * P, Nk, D, 201)
    table = torch.full((B, max(P, width)), -1, dtype=torch.int32)
    table[:, :P] = _table(B, P, B * P, 25)
    start[1, 1] = 2
    length[2, 2] = 2 ** 31 - 1
    length[3, 1] = -1
    q_len = torch.tensor([rows, rows, rows, rows, rows + 3], dtype=torch.int32)
    q = _rand(B, rows + 5, N, D, seed=26, dtype=BF16).transpose(1, 2)
    ops.check_status()
    out, lse = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.1, q_len=q_len.cuda(), return_lse=True)
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    assert not out[1:].any() and (lse[1:] == -torch.inf).all()
    ref, ref_lse, size = ch.attention(q[:1], hk, hv, table[:1], start[:1], length[:1], 0.1, q_len[:1])
    _check(out[:1], lse[:1], ref, ref_lse, size, hv, 64)


def test_captured_prompts_replay_on_new_inputs():
    """Calls that take workspaces, as one graph: over two thousand tokens written, read back, a block of many rows over a wide table, one row
    over a long one, scores."""
    N, Nk, D, B, rows = 8, 2, 128, 2, 40
    start, length, P = ch.spans([[30, 800, 300, rows], [30, 64, 700, rows]], True)
    S = P * PAGE
    st, ln = start.cuda(), length.cuda()
    table = torch.full((B, 4000), -1, dtype=torch.int32)
    table[:, :P] = _table(B, P, B * P, 27)
    tab = table.cuda()
    cache = ops.cache_alloc(B * P, Nk, D, "cuda")
    slots = torch.stack([ch.slots_of(table[b], torch.arange(S)) for b in range(B)]).int().cuda()
    k, v = (torch.zeros(B, S, Nk, D, dtype=BF16, device="cuda").transpose(1, 2) for _ in range(2))
    q = torch.zeros(B, rows, N, D, dtype=BF16, device="cuda").transpose(1, 2)
    ops.status_word("cuda")

    def run():
        ops.cache_write(k, v, cache, slots)
        ck, _ = ops.cache_read(cache, slots)
        return (ck, ops.cache_attention(q, cache, tab, st, ln, 0.1), ops.cache_attention(q[:, :, :1], cache, tab, st, ln, 0.1),
                ops.cache_doc_scores(q[:, :, :2], cache, tab, st, ln, 0.1, 800)[0])
    with torch.cuda.stream(torch.cuda.Stream()):
        run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for i in range(4):
        nk, nv = (_rand(B, S, Nk, D, seed=50 + 2 * i + j, dtype=BF16) for j in range(2))
        nq = _rand(B, rows, N, D, seed=60 + i, dtype=BF16).transpose(1, 2)
        for dst, src in ((k, nk.transpose(1, 2)), (v, nv.transpose(1, 2)), (q, nq)):
            dst.copy_(src)
        graph, (ck, many, one, mass) = graphs[i % 2]
        graph.replay()
        assert torch.equal(ck.double().cpu(), ch.held(nk).transpose(1, 2))
        hk, hv = (torch.zeros(B * P * PAGE, Nk, D, dtype=torch.float64) for _ in range(2))
        hk[slots.cpu().long().flatten()], hv[slots.cpu().long().flatten()] = ch.held(nk).flatten(0, 1), ch.held(nv).flatten(0, 1)
        for got, x in ((many, nq), (one, nq[:, :, :1])):
            ref, _, size = ch.attention(x, hk, hv, table, start, length, 0.1)
            _check(got, None, ref, None, size, hv, 3 * P + 8)
        assert torch.allclose(mass.double().cpu(), ch.doc_mass(nq[:, :, :2], hk, table, start, length, 0.1), rtol=1e-3, atol=1e-6)
    ops.check_status()


def test_calls_with_workspaces_on_two_streams_at_once():
    N, Nk, D, rows = 8, 2, 128, 40
    start, length, P = ch.spans([[30, 900, rows]], True)
    table = torch.full((1, 4000), -1, dtype=torch.int32)
    table[:, :P] = torch.arange(P, dtype=torch.int32)
    T = P * PAGE
    slots = torch.arange(T, dtype=torch.int32)[None].repeat(1, 2)  # every slot twice: the second counts
    data = []
    for i in range(2):
        k, v = (_rand(1, 2 * T, Nk, D, seed=70 + 2 * i + j, dtype=BF16) for j in range(2))
        q = _rand(1, rows, N, D, seed=80 + i, dtype=BF16).transpose(1, 2)
        data.append((k, v, q, ops.cache_alloc(P, Nk, D, "cuda"), k.cuda().transpose(1, 2), v.cuda().transpose(1, 2), q.cuda()))
    st, ln, tab, sl = start.cuda(), length.cuda(), table.cuda(), slots.cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, (_, _, _, cache, k, v, q) in enumerate(data):
            with torch.cuda.stream(streams[i]):
                ops.cache_write(k, v, cache, sl)
                outs[i].append((ops.cache_attention(q, cache, tab, st, ln, 0.1), ops.cache_attention(q[:, :, :1], cache, tab, st, ln, 0.1)))
    torch.cuda.synchronize()
    for i, (k, v, q, *_) in enumerate(data):
        hk, hv = ch.held(k)[0, T:], ch.held(v)[0, T:]
        for n, x in enumerate((q, q[:, :, :1])):
            for out in outs[i]:
                assert torch.equal(out[n], outs[i][0][n])
            ref, _, size = ch.attention(x, hk, hv, table, start, length, 0.1)
            _check(outs[i][0][n], None, ref, None, size, hv, 3 * P + 8)
    ops.check_status()


def test_very_many_heads():
    Nk, D, S = 300, 64, 5
    k, v = (_rand(1, S, Nk, D, seed=90 + i, dtype=BF16) for i in range(2))
    cache = ops.cache_alloc(2, Nk, D, "cuda")
    slots = torch.tensor([[70, 3, -1, 127, 64]], dtype=torch.int32)
    ops.cache_write(k.cuda().transpose(1, 2), v.cuda().transpose(1, 2), cache, slots.cuda())
    gk, gv = ops.cache_read(cache, slots.cuda(), F32)
    keep = (slots >= 0)[:, None, :, None]
    assert torch.equal(gk.double().cpu(), torch.where(keep, ch.held(k).transpose(1, 2), 0.0))
    assert torch.equal(gv.double().cpu(), torch.where(keep, ch.held(v).transpose(1, 2), 0.0))
    ops.check_status()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [9, 40])
def test_pages_of_which_only_a_part_is_in_a_block(D, rows):
    """Blocks in the first half of a page, in the second, across the middle, in single tokens at either end; NaN next to them."""
    N, Nk = 8, 2
    spans = [(0, 32), (96, 32), (128, 1), (191, 1), (220, 8), (256 + 31, 1), (320 + 32, 1), (384, 63), (449, 63), (576, 100 + rows)]
    start, length = (torch.tensor([[s[i] for s in spans]], dtype=torch.int32) for i in (0, 1))
    P = 14
    cache, hk, hv = _filled(P, Nk, D, 211)
    inside = torch.cat([torch.arange(a, a + n) for a, n in spans])
    table = _table(1, P, P, 28)
    at = ch.slots_of(table[0], inside)[None].int().cuda()
    k, v = ops.cache_read(cache, at, F32)
    cache.fill_(255)
    ops.cache_write(k, v, cache, at)
    q = _rand(1, rows, N, D, seed=29, dtype=BF16).transpose(1, 2)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, 0.1)
    for tab in (table, _wide(table)):
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), 0.1, return_lse=True)
        _check(out, lse, ref, ref_lse, size, hv, 64)
    ops.check_status()


@pytest.mark.parametrize("docs,Nk", [(4, 2), (32, 8), (32, 1), (33, 2), (5, 12)])
def test_scores_of_a_document_with_nan(docs, Nk):
    """NaN in one head's keys of one document: NaN in all documents of that head's rows (a softmax over them), in the prompt's logits,
    and nowhere else; with and without a kernel that merges."""
    N, D, R, B = 2 * Nk, 64, 2, 3
    start, length, P = ch.spans([[5] + [17] * docs + [9]] * B, False)
    cache, hk, hv = _filled(B * P, Nk, D, 221)
    table = _table(B, P, B * P, 30)
    q = _rand(B, R, N, D, seed=31, dtype=BF16).transpose(1, 2)
    args = (cache, table.cuda(), start.cuda(), length.cuda(), 0.1, 17)
    ref = ch.doc_mass(q, hk, table, start, length, 0.1)
    mass, out = ops.cache_doc_scores(q.cuda(), *args)
    assert torch.allclose(mass.double().cpu(), ref, rtol=1e-4) and torch.allclose(out.double().cpu(), ref.mean((1, 2)) / 0.05, rtol=1e-4)
    at = ch.slots_of(table[1], start[1, 2:3].long() + 3)[None].int().cuda()
    k, v = ops.cache_read(cache, at, F32)
    k[0, 0, 0, 7] = torch.nan
    ops.cache_write(k, v, cache, at)
    bad, bad_out = ops.cache_doc_scores(q.cuda(), *args)
    assert bad[1, :2].isnan().all() and bad_out[1].isnan().all()
    assert torch.equal(bad[1, 2:], mass[1, 2:])
    for b in (0, 2):
        assert torch.equal(bad[b], mass[b]) and torch.equal(bad_out[b], out[b])
    ops.check_status()


@pytest.mark.parametrize("N,Nk,D", [(32, 8, 128), (16, 8, 64), (8, 8, 128)])
@pytest.mark.parametrize("rows", [40, 70])
def test_query_blocks_of_a_batch(N, Nk, D, rows):
    """So many prompts that each has a CTA of the tcgen05 kernel for a KV head: one tile of rows, two, and more; no parts to join."""
    B = 40
    g = torch.Generator().manual_seed(6)
    lens = [torch.randint(0, 130, (3,), generator=g).tolist() + [rows + b % 3] for b in range(B)]
    start, length, P = ch.spans(lens, True)
    cache, hk, hv = _filled(B * P, Nk, D, 231)
    table = _table(B, P, B * P, 32)
    q_len = torch.tensor([rows - b % 5 if b % 7 else 0 for b in range(B)], dtype=torch.int32)
    start[11, 2] = start[11, 1] + length[11, 1] - 1 if lens[11][1] else -1  # malformed
    q = _rand(B, rows, N, D, seed=33, dtype=BF16).transpose(1, 2)
    ops.check_status()
    out, lse = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), D ** -0.5, q_len=q_len.cuda(), return_lse=True)
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    q_len[11] = 0
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, D ** -0.5, q_len)
    _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)


@pytest.mark.parametrize("dtype,N,Nk,D,T", [(BF16, 4, 1, 64, 2500), (F32, 4, 1, 64, 1100), (BF16, 2, 2, 128, 1300)])
def test_a_whole_sequence_at_once(dtype, N, Nk, D, T):
    """As many rows as there are tokens: each sees those up to its own."""
    P = -(-T // PAGE)
    cache, hk, hv = _filled(P, Nk, D, 241, dtype)
    table = _table(1, P, P, 34)
    start, length = torch.zeros(1, 1, dtype=torch.int32), torch.full((1, 1), T, dtype=torch.int32)
    q = _rand(1, T, N, D, seed=35, dtype=dtype).transpose(1, 2)
    at = ch.slots_of(table[0], torch.arange(T))
    k, v = (x[at].repeat_interleave(N // Nk, 1).transpose(0, 1) for x in (hk, hv))
    x = q[0].double() @ k.transpose(1, 2) * 0.1
    late = torch.ones(T, T).triu(1).bool()
    ref_lse = torch.logsumexp(x.masked_fill(late, -torch.inf), -1)[None]
    ref = (torch.softmax(x.masked_fill(late, -torch.inf), -1) @ v).transpose(0, 1)[None]
    size = (q[0].double().abs() @ k.abs().transpose(1, 2) * 0.1).amax()
    for tab in (table, _wide(table)):
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), 0.1, return_lse=True)
        _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
    ops.check_status()


def test_scales_next_to_the_borders_of_the_smallest_ones():
    """fp32 groups whose largest magnitude is 7 (k + 1/2) 2^-130 or up to three last places of it away: the scale's grid is that of 2^-130
    there, and a seventh of such a magnitude is no normal number."""
    k = torch.arange(0, 17, dtype=torch.float64) + 0.5
    top = torch.ldexp(7 * k, torch.tensor(-130)).float()
    top = (top.view(torch.int32)[:, None] + torch.arange(-3, 4, dtype=torch.int32)).flatten().view(F32)
    g = torch.linspace(-1, 1, 32, dtype=torch.float64)
    x = (top.double()[:, None] * g).float()
    x[:, 0] = top
    x = torch.cat([x, x.flip(-1)], -1)[None, None]  # (B, Nk, S, D)
    slots = torch.arange(x.shape[2], dtype=torch.int32)[None]
    cache = ops.cache_alloc(2, 1, 64, "cuda")
    ops.cache_write(x.cuda(), -x.cuda(), cache, slots.cuda())
    for got, src in zip(ops.cache_read(cache, slots.cuda(), F32), (x, -x)):
        assert torch.equal(got.double().cpu(), ch.held(src))
    ops.check_status()


@pytest.mark.parametrize("docs", [3, 40, 200])
def test_scores_of_a_prompt_with_a_malformed_block(docs):
    """One malformed block, whichever it is, leaves its whole prompt without documents; a page that does not exist only takes its own tokens
    away.  Each is reported by itself; the other prompts have their masses and logits.  (Prompts whose CTAs make the logits
    themselves, prompts that are merged, more documents than a CTA has threads.)"""
    N, Nk, D, R, most = 4, 2, 64, 2, 70
    lens = [9] + [most - (i % 7) for i in range(docs)] + [12]
    start, length, P = ch.spans([lens], True)
    broken = {
        "none": None,
        "a document that runs into the next one": lambda st, ln: st[docs].fill_(int(st[docs - 1] + ln[docs - 1]) - 1),
        "a document that is too long": lambda st, ln: ln[2].fill_(most + 1),
        "the last document runs into the query block": lambda st, ln: st[-1].fill_(int(st[-2] + ln[-2]) - 1),
        "an instruction block of negative length": lambda st, ln: ln[0].fill_(-1),
        "an instruction block in front of the first slot": lambda st, ln: st[0].fill_(-1),
        "an instruction block that runs into the first document": lambda st, ln: ln[0].fill_(int(st[1]) + 1),
        "a query block behind the page table": lambda st, ln: st[-1].fill_(P * PAGE - 11),
        "no page": "page",
    }
    B = len(broken)
    pool = B * P + 1
    cache, hk, _ = _filled(pool, Nk, D, 251)
    table = _table(B, P, pool, 36)
    q = _rand(B, R, N, D, seed=37, dtype=BF16).transpose(1, 2)
    st, ln, tab = start.repeat(B, 1), length.repeat(B, 1), table.clone()
    seen_st, seen_ln = st.clone(), ln.clone()  # what is left to be seen
    for b, (name, how) in enumerate(broken.items()):
        if how == "page":  # of the second document's two pages the last one
            tab[b, int(start[0, 2]) // PAGE + 1] = pool
            seen_ln[b, 2] = PAGE
        elif how is not None:
            how(st[b], ln[b])
            seen_ln[b] = 0
    ref = ch.doc_mass(q, hk, table, seen_st, seen_ln, 0.2)
    assert bool((ref[0] > 0).all()) and bool((ref[-1] > 0).all())
    size = float(torch.einsum("bnrd,snd->bnrs", q.double().abs(), hk.abs().repeat_interleave(N // Nk, 1)).max()) * 0.2
    rel = 2 * size * 24 * 2.0 ** -23 + 64 * 2.0 ** -23  # (as in test_document_scores)
    assert rel < 1 / (4 * docs)  # (a document too many or too few shows)
    ops.check_status()

    def check(of):
        mass, logits = ops.cache_doc_scores(q[of].cuda(), cache, tab[of].cuda(), st[of].cuda(), ln[of].cuda(), 0.2, most)
        assert torch.allclose(mass.double().cpu(), ref[of], rtol=rel, atol=0)
        assert torch.allclose(logits.double().cpu(), ref[of].mean((1, 2)) / 0.05, rtol=2 * rel, atol=0)
    for b in range(B):
        check(slice(b, b + 1))
        if b == 0:
            ops.check_status()
        else:
            with pytest.raises(ValueError, match="of a call on the cache"):
                ops.check_status()
    check(slice(0, B))
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()


def test_a_document_behind_one_that_is_too_long_only():
    """Overlap and length each alone: a document longer than max_block_len that touches no other."""
    N, Nk, D = 4, 2, 64
    start, length, P = ch.spans([[3, 70, 60, 9]], True, gap=PAGE)
    cache, hk, _ = _filled(P, Nk, D, 261)
    table = _table(1, P, P, 38)
    q = _rand(1, 1, N, D, seed=39, dtype=BF16).transpose(1, 2)
    args = (q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.2)
    ops.check_status()
    mass, logits = ops.cache_doc_scores(*args, 70)
    ops.check_status()
    assert torch.allclose(mass.double().cpu(), ch.doc_mass(q, hk, table, start, length, 0.2), rtol=1e-4)
    mass, logits = ops.cache_doc_scores(*args, 69)
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    assert not mass.any() and not logits.any()


def _attention_of_long(q, hk, hv, table, start, length, scale, q_len):
    """ch.attention for long prompts of many rows (a prompt's rows together, on the GPU); entries of -1 in the table do not exist."""
    B, N, R, D = q.shape
    outs, lses, sizes = [], [], []
    for b in range(B):
        rows, slot = int(q_len[b]), torch.cat([torch.arange(a, a + n) for a, n in zip(start[b].tolist(), length[b].tolist())])
        slot = slot[table[b][slot // PAGE] >= 0]
        at = ch.slots_of(table[b], slot)
        k, v = (x[at].repeat_interleave(N // x.shape[1], 1).transpose(0, 1).cuda() for x in (hk, hv))
        own = int(start[b, -1] + length[b, -1]) - rows + torch.arange(rows)
        qq = q[b, :, :rows].double().cuda()
        x = (qq @ k.transpose(1, 2) * scale).masked_fill((slot > own[:, None]).cuda(), -torch.inf)
        pad = (0, R - rows)
        outs.append(torch.nn.functional.pad((torch.softmax(x, -1) @ v).transpose(0, 1), (0, 0, 0, 0) + pad))
        lses.append(torch.nn.functional.pad(torch.logsumexp(x, -1), pad, value=-torch.inf))
        sizes.append((qq.abs() @ k.abs().transpose(1, 2) * scale).amax())
    return torch.stack(outs).cpu(), torch.stack(lses).cpu(), torch.stack(sizes).cpu()


@pytest.mark.parametrize("dtype,N,Nk,D,R,pages,B", [
    (BF16, 4, 2, 64, 1, 300, 1800), (BF16, 4, 2, 128, 2, 300, 1800), (BF16, 8, 2, 128, 2, 300, 1800), (BF16, 6, 2, 64, 5, 300, 1200),
    (F32, 4, 2, 64, 1, 300, 1200), (F32, 2, 1, 64, 8, 300, 2400), (F32, 6, 2, 128, 2, 300, 1200),
    (BF16, 4, 2, 128, 20, 700, 600), (BF16, 4, 2, 64, 70, 700, 600),
    # fewer prompts: two long shares each, joined by a cluster (few rows) or a kernel (many), or ten, joined by a kernel
    (BF16, 4, 2, 64, 1, 300, 111), (F32, 4, 2, 128, 3, 300, 74), (BF16, 4, 2, 128, 20, 1100, 37), (BF16, 4, 2, 64, 70, 1100, 37), (BF16, 2, 1, 64, 1, 1500, 44)])
def test_shares_of_more_pages_than_a_cta_knows_of_at_a_time(dtype, N, Nk, D, R, pages, B):
    """Shares of pages that are looked at in several goes, first so many prompts that each is one share: blocks that end and begin where those do,
    a whole go without a token, prompts far shorter than the table, a page that does not exist.  (The prompts are 10 in turn.)"""
    T, at = pages * PAGE, lambda page, more=0: page * PAGE + more
    go = 256 if pages > 300 else 128
    prompts = [  # (start, length) of three blocks
        [(0, 50), (at(1), at(pages - 4)), (at(pages - 2), 2 * PAGE)],
        [(0, at(go)), (at(go), at(go)), (at(2 * go), R + 1)],
        [(0, at(go, -1)), (at(go, 1), 3), (at(2 * go, -1), R + 2)],
        [(0, 1), (at(2 * go), 1), (at(pages - 2, 3), R + 40)],          # a go with nothing
        [(at(2 * go, 5), 1), (at(2 * go, 6), 0), (at(2 * go + 1), R)],  # nothing before the last go
        [(0, 5), (7, 0), (9, R)],
        [(0, at(go)), (at(go), 0), (at(go), R + 63)],
        [(3, at(1)), (at(5), at(go, 17)), (T - R, R)],
        [(1, 31), (at(go, 32), 32), (T - R - 9, R + 9)],
        [(0, T - 70), (T - 70, 0), (T - 70, 70)],
    ]
    start, length = (torch.tensor([[s[i] for s in p] for p in prompts], dtype=torch.int32) for i in (0, 1))
    K = len(prompts)
    cache, hk, hv = _filled(pages, Nk, D, 271, dtype)
    table = _table(1, pages, pages, 40).repeat(K, 1)
    q_len = torch.tensor([R - b % 3 if R > 3 else R for b in range(K)], dtype=torch.int32)
    q = _rand(K, R, N, D, seed=41, dtype=dtype).transpose(1, 2)
    ref, ref_lse, size = _attention_of_long(q, hk, hv, table, start, length, D ** -0.5, q_len)
    rep = lambda x: x.repeat(-(-B // K), *[1] * (x.dim() - 1))[:B].cuda()
    args = (rep(q), cache, rep(table), rep(start), rep(length), D ** -0.5)
    ops.check_status()
    out, lse = ops.cache_attention(*args, q_len=rep(q_len), return_lse=True)
    ops.check_status()
    _check(out[:K], lse[:K], ref, ref_lse, size, hv, 3 * pages + 8)
    assert torch.equal(out, rep(out[:K])) and torch.equal(lse, rep(lse[:K]))
    # the last page of one prompt does not exist, nor a page of another's second go
    tab, kept = args[2].clone(), table[[0, 1]].clone()
    tab[K, pages - 1], kept[0, pages - 1] = pages, -1
    tab[K + 1, go + 7], kept[1, go + 7] = -5, -1
    out2, lse2 = ops.cache_attention(args[0], cache, tab, *args[3:], q_len=rep(q_len), return_lse=True)
    with pytest.raises(ValueError, match="of a call on the cache"):
        ops.check_status()
    same = (torch.arange(B) - K) // 2 != 0
    assert torch.equal(out2[same.cuda()], out[same.cuda()]) and torch.equal(lse2[same.cuda()], lse[same.cuda()])
    ref, ref_lse, size = _attention_of_long(q[:2], hk, hv, kept, start[:2], length[:2], D ** -0.5, q_len[:2])
    _check(out2[K:K + 2], lse2[K:K + 2], ref, ref_lse, size, hv, 3 * pages + 8)
    # NaN in the value of the last slot but one, in one head and 32 channels: in the rows that see it, and in nothing else of theirs
    at = ch.slots_of(table[0], torch.tensor([T - 2]))[None].int().cuda()
    k1, v1 = ops.cache_read(cache, at, F32)
    v1[:, 0, 0, 5] = torch.nan
    ops.cache_write(k1, v1, cache, at)
    bad, bad_lse = ops.cache_attention(*args, q_len=rep(q_len), return_lse=True)
    ends, i = (start + length)[:, -1:], torch.arange(R)[None]
    sees = (start[:, -1:] <= T - 2) & (ends - q_len[:, None] + i >= T - 2) & (i < q_len[:, None])  # (K, R)
    want = out[:K].clone()
    want[:, :, :N // Nk, :32] = torch.where(sees[:, :, None, None].cuda(), torch.nan, want[:, :, :N // Nk, :32])
    assert bool(sees.any()) and torch.equal(bad_lse, lse)
    assert torch.equal(bad[:K].isnan(), want.isnan()) and torch.equal(bad[:K].nan_to_num(), want.nan_to_num())
    assert torch.equal(bad.nan_to_num(), rep(bad[:K]).nan_to_num())
    ops.check_status()


@pytest.mark.parametrize("dtype,N,Nk,D,T", [(BF16, 4, 1, 64, 40000), (BF16, 8, 2, 128, 18000), (F32, 2, 1, 64, 20000)])
def test_a_long_sequence_at_once(dtype, N, Nk, D, T):
    """As many rows as tokens, longer than a CTA knows the pages of at a time; rows here and there against 64 bits."""
    P = -(-T // PAGE)
    cache, hk, hv = _filled(P, Nk, D, 281, dtype)
    table = _table(1, P, P, 42)
    start, length = torch.zeros(1, 1, dtype=torch.int32), torch.full((1, 1), T, dtype=torch.int32)
    q = _rand(1, T, N, D, seed=43, dtype=dtype).transpose(1, 2)
    out, lse = ops.cache_attention(q.cuda(), cache, table.cuda(), start.cuda(), length.cuda(), 0.1, return_lse=True)
    at = ch.slots_of(table[0], torch.arange(T))
    k, v = (x[at].repeat_interleave(N // Nk, 1).transpose(0, 1).cuda() for x in (hk, hv))
    rows = torch.cat([torch.arange(0, T, 997), torch.tensor([63, 64, 127, 8191, 8192, 16383, 16384, T - 2, T - 1])]).cuda()
    qq = q[0].cuda()[:, rows].double()
    x = (qq @ k.transpose(1, 2) * 0.1).masked_fill(torch.arange(T, device="cuda") > rows[:, None], -torch.inf)
    ref, ref_lse = (torch.softmax(x, -1) @ v).transpose(0, 1)[None], torch.logsumexp(x, -1)[None]
    size = (qq.abs() @ k.abs().transpose(1, 2) * 0.1).amax()
    _check(out[:, rows], lse[:, :, rows], ref.cpu(), ref_lse.cpu(), size, hv, 3 * P + 8)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    ops.check_status()


@pytest.mark.parametrize("S,different", [(2049, 40), (4096, 4096), (20000, 5000)])
@pytest.mark.parametrize("step", [1, 64, 8191, 1048573])
def test_of_tokens_with_the_same_slot_the_last_one_is_kept_in_a_large_pool(S, different, step):
    """A pool so much larger than the call that the tokens of its slots are looked up by hash; slots side by side, page by page, far apart."""
    Nk, D, pool = 1, 64, 2 ** 18 + 1000
    n_slots = pool * PAGE
    c = _lib.Cache(64, pool, Nk, D)
    assert _lib.lib().brk_cache_write_workspace_bytes(c, 1, S) < 4 * n_slots
    k, v = (_rand(1, S, Nk, D, seed=i, dtype=BF16) for i in (0, 1))
    g = torch.Generator().manual_seed(S)
    slots = (torch.randint(0, different, (1, S), generator=g) * step % n_slots).int()
    slots[0, ::17] = -1
    slots[0, 5::97] = n_slots + 3
    last = {s: i for i, s in enumerate(slots[0].tolist()) if 0 <= s < n_slots}
    cache = ops.cache_alloc(pool, Nk, D, "cuda")
    ops.check_status()
    ops.cache_write(k.transpose(1, 2).cuda(), v.transpose(1, 2).cuda(), cache, slots.cuda())
    with pytest.raises(ValueError, match="slot lies outside the cache"):
        ops.check_status()
    at, tok = torch.tensor(list(last), dtype=torch.int32)[None], torch.tensor(list(last.values()))
    for got, x in zip(ops.cache_read(cache, at.cuda(), F32), (k, v)):
        assert torch.equal(got[0].transpose(0, 1).double().cpu(), ch.held(x[0, tok]))
    pages = torch.ones(pool, dtype=torch.bool)
    pages[at[0].long() // PAGE] = False
    assert not cache[pages.cuda()].any()
    others = torch.ones(n_slots, dtype=torch.bool)
    others[at[0].long()] = False
    rest = (others.view(pool, PAGE) & ~pages[:, None]).view(-1).nonzero().T.int().cuda()
    assert not any(x.any() for x in ops.cache_read(cache, rest, F32))
    ops.check_status()


def test_gradients_are_refused_and_not_dropped():
    cache, _, _ = _filled(2, 2, 64, 301)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    x, one = (torch.ones(1, n, 1, 64, dtype=BF16, device="cuda") for n in (4, 2))
    spans = z(1, 1), torch.arange(3, dtype=torch.int32, device="cuda")[None], z(1, 3) + 1  # the page table, three blocks of one token
    attend, score = lambda: ops.cache_attention(x, cache, *spans, 1.0), lambda: ops.cache_doc_scores(x, cache, *spans, 1.0, 1)
    want = attend(), score()
    before = cache.clone()
    x.requires_grad_(), one.requires_grad_()
    for call in (attend, score, lambda: ops.cache_write(one, one, cache, z(1, 1))):
        with pytest.raises(NotImplementedError, match="inference-only"):
            call()
    assert torch.equal(cache, before)
    with torch.no_grad():
        got = attend(), score()
        ops.cache_write(one, one, cache, z(1, 1))
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    assert not torch.equal(cache, before)
    ops.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 3, 5, 20])
@pytest.mark.parametrize("scale", [1e-12, 1e-30, 1.2e-38])
def test_queries_of_zeros_and_scales_next_to_nothing(dtype, rows, scale):
    """Every slot counts the same: the mean of the values, the logarithm of their number, documents by their tokens."""
    N, Nk, D = 4, 2, 64
    start, length, P = ch.spans([[5, 64, 1, 100, rows + 30], [1, 63, 65, 0, rows]], False, gap=3)
    cache, hk, hv = _filled(2 * P, Nk, D, 311, dtype)
    table = _table(2, P, 2 * P, 44)
    q = _rand(2, rows, N, D, seed=45, dtype=dtype).transpose(1, 2).contiguous()
    q[:, 1] = 0
    q[:, 2] = torch.finfo(dtype).tiny / 4
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, scale)
    for tab in (table, _wide(table)):
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), scale, return_lse=True)
        _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
    mass, logits = ops.cache_doc_scores(q[:, :, :3].cuda(), cache, table.cuda(), start.cuda(), length.cuda(), scale, 100)
    want = ch.doc_mass(q[:, :, :3], hk, table, start, length, scale)
    assert torch.allclose(mass.double().cpu(), want, rtol=2.0 ** -16, atol=0)  # (64 accumulations of 2^-23, as in test_document_scores)
    assert torch.allclose(logits.double().cpu(), want.mean((1, 2)) / 0.05, rtol=2.0 ** -16, atol=0)
    ops.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 5, 20])
@pytest.mark.parametrize("e,scale", [(114, 1.0), (112, 4.0), (114, 1e-3), (60, 1.0), (-100, 1.0)])
def test_queries_as_large_as_they_may_be(dtype, rows, e, scale):
    """Largest magnitude next to 2^e, of keys that make ordinary logits of them."""
    N, Nk, D = 4, 2, 64
    start, length, P = ch.spans([[5, 64, 1, 100, rows + 30]], False)
    k, v = (_rand(P * PAGE, Nk, D, seed=321 + i, dtype=F32) for i in (0, 1))
    k, v = (k.clamp(-4, 4) * 2.0 ** -e / scale).to(dtype), v.to(dtype)
    cache = ops.cache_alloc(P, Nk, D, "cuda")
    ops.cache_write(*(x[None].transpose(1, 2).cuda() for x in (k, v)), cache, torch.arange(P * PAGE, dtype=torch.int32, device="cuda")[None])
    hk, hv, table = ch.held(k), ch.held(v), torch.arange(P, dtype=torch.int32)[None]
    q = _rand(1, rows, N, D, seed=46, dtype=F32)
    q = (q / q.abs().max() * 2.0 ** e * 0.99).to(dtype).transpose(1, 2)
    ref, ref_lse, size = ch.attention(q, hk, hv, table, start, length, scale)
    for tab in (table, _wide(table)):
        out, lse = ops.cache_attention(q.cuda(), cache, tab.cuda(), start.cuda(), length.cuda(), scale, return_lse=True)
        _check(out, lse, ref, ref_lse, size, hv, 3 * P + 8)
    mass, _ = ops.cache_doc_scores(q[:, :, :2].cuda(), cache, table.cuda(), start.cuda(), length.cuda(), scale, 100)
    want = ch.doc_mass(q[:, :, :2], hk, table, start, length, scale)
    assert torch.allclose(mass.double().cpu(), want, rtol=2 * float(size.max()) * 24 * 2.0 ** -23 + 2.0 ** -17, atol=0)
    ops.check_status()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_properties_of_what_the_kernels_hold(dtype, D):
    """Read back, values are exact in bf16, half a step of their scale off at most, and held as the same bytes when written again."""
    Nk, pool = 3, 8
    g = torch.Generator().manual_seed(9)
    x = [(torch.randn(pool * PAGE, Nk, D, generator=g) * torch.exp(8 * torch.randn(pool * PAGE, Nk, 1, generator=g))).to(dtype) for _ in range(2)]
    every = torch.arange(pool * PAGE, dtype=torch.int32, device="cuda")[None]
    caches = [ops.cache_alloc(pool, Nk, D, "cuda") for _ in range(3)]
    ops.cache_write(*(t[None].transpose(1, 2).cuda() for t in x), caches[0], every)
    wide, narrow = (ops.cache_read(caches[0], every, t) for t in (F32, BF16))
    for w, n, t in zip(wide, narrow, x):
        assert torch.equal(w, n.float())
        half = ch.scales(t).repeat_interleave(32, -1) / 2
        assert bool(((w[0].transpose(0, 1).double().cpu() - t.double()).abs() <= half).all())
    for held, c in zip((wide, narrow), caches[1:]):
        ops.cache_write(*held, c, every)
        assert torch.equal(c, caches[0])
    ops.check_status()
