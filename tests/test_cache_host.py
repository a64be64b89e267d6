"""The 4-bit cache without a GPU: refusals of the C ABI and the properties of what is held."""
import ctypes as C

import pytest
import torch

from blockrank_b200 import _lib, ops
from tests import cache_helpers as ch


def _cache(n_pages=4, Nk=2, D=64, ptr=64):
    return _lib.Cache(ptr, n_pages, Nk, D)


def _view(D=64, ptr=64):
    return _lib.View(ptr, 8 * D, D, 2 * D)


def test_sizes():
    L = _lib.lib()
    assert L.brk_cache_page_bytes(1, 64) == 64 * 72 and L.brk_cache_page_bytes(8, 128) == 8 * 64 * 144
    assert L.brk_cache_page_bytes(1, 96) == 0 and L.brk_cache_page_bytes(0, 64) == 0
    c = _cache()
    assert L.brk_cache_write_workspace_bytes(C.byref(c), 8, 256) == 0
    assert L.brk_cache_write_workspace_bytes(C.byref(c), 8, 257) == 4 * 64 * 4
    assert L.brk_cache_attn_workspace_bytes(None) == 0 and L.brk_cache_doc_scores_workspace_bytes(None) == 0


@pytest.mark.parametrize("change,code", [
    (dict(cache=None), -1), (dict(ptr=0), -1), (dict(ptr=72), -1), (dict(D=96), -2), (dict(n_pages=0), -1), (dict(Nk=0), -1),
    (dict(n_pages=2 ** 25), -1), (dict(dtype=2), -2), (dict(slots=None), -1), (dict(S=0), -1), (dict(B=2 ** 16, S=2 ** 16), -1),
    (dict(view=0), -1), (dict(view=8), -1), (dict(S=2049), -3)])
def test_refusals_of_write(change, code):
    """(every one of them is refused in front of any launch)"""
    L = _lib.lib()
    a = dict(ptr=64, n_pages=4, Nk=2, D=64, dtype=0, B=1, S=3, slots=64, view=64, cache=True)
    a.update(change)
    c = _cache(a["n_pages"], a["Nk"], a["D"], a["ptr"])
    v = _view(ptr=a["view"])
    args = (a["dtype"], C.byref(c) if a["cache"] else None, C.byref(v), C.byref(v), a["B"], a["S"], a["slots"])
    assert L.brk_cache_write(*args, None, 0, None, None) == code, L.brk_last_error()
    if code != -3:
        assert L.brk_cache_read(*args, None, None) == code, L.brk_last_error()


def _attn(**change):
    p = _lib.CacheAttnParams()
    p.dtype, p.B, p.N, p.Lq, p.M, p.P, p.scale = 0, 1, 4, 1, 1, 1, 1.0
    p.cache, p.q, p.o = _cache(), _view(), _view()
    p.page_table = p.blk_start = p.blk_len = 64
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), -2), (dict(B=0), -1), (dict(N=5), -1), (dict(Lq=0), -1), (dict(M=0), -1), (dict(P=0), -1), (dict(P=2 ** 25), -1),
    (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(page_table=None), -1),
    (dict(blk_len=None), -1), (dict(B=40000), -2), (dict(B=30000, Lq=2 ** 16), -1), (dict(q=_view(ptr=8)), -1), (dict(o=_view(ptr=0)), -1),
    (dict(cache=_cache(D=32)), -2)])
def test_refusals_of_attention(change, code):
    L = _lib.lib()
    p = _attn(**change)
    assert L.brk_cache_attn(C.byref(p), None, 0, None) == code, L.brk_last_error()
    assert L.brk_cache_attn(None, None, 0, None) == -1


def test_a_workspace_that_is_too_small_is_refused():
    L = _lib.lib()
    p = _attn(P=4096)
    need = L.brk_cache_attn_workspace_bytes(C.byref(p))
    assert need > 0 and L.brk_cache_attn(C.byref(p), 64, need - 1, None) == -3


@pytest.mark.parametrize("change,code", [
    (dict(M=2), -1), (dict(R=65), -1), (dict(max_block_len=0), -1), (dict(temperature=0.0), -1), (dict(doc_mass=None), -1), (dict(N=3), -1), (dict(M=40, P=40), -3)])
def test_refusals_of_scores(change, code):
    L = _lib.lib()
    p = _lib.CacheScoreParams()
    p.dtype, p.B, p.N, p.R, p.M, p.P, p.max_block_len, p.scale, p.temperature = 0, 1, 4, 1, 3, 1, 64, 1.0, 0.05
    p.cache, p.q = _cache(), _view()
    p.page_table = p.blk_start = p.blk_len = p.doc_mass = 64
    for k, v in change.items():
        setattr(p, k, v)
    assert L.brk_cache_doc_scores(C.byref(p), None, 0, None) == code, L.brk_last_error()


def test_cpu_tensors_are_refused():
    i = torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(1, 1, 1, 64)
    c = torch.zeros(1, 1, 64 * 72, dtype=torch.uint8)
    for call in (lambda: ops.cache_alloc(1, 1, 64, "cpu"), lambda: ops.cache_write(x, x, c, i), lambda: ops.cache_read(c, i),
                 lambda: ops.cache_attention(x, c, i, i, i, 1.0), lambda: ops.cache_doc_scores(x, c, i, i, i, 1.0, 1)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()


def test_what_is_held():
    """Held values are exact in bf16, held as themselves when written again, and half a step of their scale off at most."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 3, 128, generator=g) * torch.exp(8 * torch.randn(500, 3, 1, generator=g))
    h = ch.held(x)
    assert torch.equal(h, h.float().double()) and torch.equal(h, h.bfloat16().double())
    assert torch.equal(ch.held(h), h)
    s = ch.scales(x).repeat_interleave(32, -1)
    assert bool(((h - x.double()).abs() <= s / 2 + 1e-300).all())


@pytest.mark.parametrize("dtype,N,Nk,D,Lq,tokens,B", [
    (0, 32, 8, 128, 131072, 131072, 1), (0, 32, 8, 128, 32768, 32768, 1), (0, 32, 8, 128, 4096, 131072, 1), (1, 32, 8, 128, 4096, 131072, 1),
    (1, 8, 8, 64, 65536, 65536, 1), (0, 128, 1, 128, 1, 2 ** 22, 1), (0, 32, 8, 128, 1, 131072, 1024), (0, 32, 8, 128, 48, 2 ** 24, 64)])
def test_workspaces_do_not_grow_with_the_call(dtype, N, Nk, D, Lq, tokens, B):
    """Whole sequences, long caches, many prompts: parts of 8 x 148 CTAs of 256 rows at most (include/blockrank_b200.h)."""
    view = _lib.View(64, Lq * N * D, D, N * D)
    p = _attn(dtype=dtype, N=N, Lq=Lq, B=B, P=-(-tokens // 64), cache=_cache(2 ** 18, Nk, D), q=view, o=view)
    need = _lib.lib().brk_cache_attn_workspace_bytes(C.byref(p))
    assert need <= 8 * 148 * 256 * (4 * D + 8), need


@pytest.mark.parametrize("tokens", [2049, 4096, 4097, 100000, 2 ** 26 + 1])
def test_the_workspace_of_a_write_to_a_large_pool_goes_by_its_tokens(tokens):
    """(156 million slots of 8 heads of 128 are a GPU's memory: 4 bytes of each were 625 MB for 2,049 tokens)"""
    for n_pages in (1, 33, 50000, 2 ** 18, 2 ** 18 + 1, 2 ** 21, 2 ** 25 - 1):
        need = _lib.lib().brk_cache_write_workspace_bytes(C.byref(_cache(n_pages)), 1, tokens)
        assert 0 < need <= min(4 * 64 * n_pages, max(2 ** 26, 32 * tokens))


def test_tensors_that_require_a_gradient_are_refused():
    i = torch.zeros(1, 1, dtype=torch.int32)
    x, c = torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 64 * 72, dtype=torch.uint8)
    p = x.clone().requires_grad_()
    calls = (lambda g: ops.cache_write(g, x, c, i), lambda g: ops.cache_write(x, g, c, i), lambda g: ops.cache_attention(g, c, i, i, i, 1.0),
             lambda g: ops.cache_attention(x, c, i, i, i, 1.0, out=g), lambda g: ops.cache_doc_scores(g, c, i, i, i, 1.0, 1))
    for call in calls:
        for t in (p, p * 2):
            with pytest.raises(NotImplementedError, match="inference-only"):
                call(t)
            with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors"):  # (the next refusal: there is no GPU)
                call(t)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="inference-only"):
        ops.cache_attention(torch.autograd.forward_ad.make_dual(x, x), c, i, i, i, 1.0)
