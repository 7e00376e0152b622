"""The serving operators on the GPU against plain 64-bit implementations: appending to a paged
cache with norm and rotation, attention of one new token over it, log probabilities.

Tolerances count roundings.  e(t) = finfo(t).eps / 2 is half a step of type t relative to the
value; u = 2^-24 the same for fp32.
* append: y = a c -+ b s takes two products and a sum in fp32 (3 u (|a c| + |b s|)), a norm in
  front multiplies both by a factor whose sum of D squares is off by at most D u and whose
  root and products add a few u: (D / 2 + 8) u in all; then one rounding e(t) |y|.
* decode: scores are off by ds = 2 D u scale sum |q k| (products of 16-bit numbers are exact in
  fp32; the sum may truncate, hence 2), the weights by that, the exponential's 4 u and 2^-16
  where a weight is held as two 16-bit parts: sum p |v| (2 ds + 2^-15) and e(t) |out|.
  lse is off by ds + 2^-20 (1 + |lse|).
* log probabilities: x - m and its exponential are off by u |x - m| + 4 u relative to a weight;
  a sum of V weights runs over at most 2^8 values in a row before it is joined: 2^-15 on the
  logarithm of the sum, and 2^-14 (1 + entropy) on the entropy, whose second sum has
  weights times |x - m|.
"""
import math

import pytest
import torch

import yirage_b200 as yr
from oracle import decode_oracle as O
from tests.util import oracle_weights
from yirage_b200 import _native as N
from yirage_b200 import llama

pytestmark = pytest.mark.gpu
F64 = torch.float64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Batch:
    """Page tables of requests with the given lengths (new tokens included) over a pool in random
    order; the pool is full of NaN wherever no request has a token."""

    def __init__(self, lengths, new=None, *, page=64, heads=2, dim=128, dtype=BF16, seed=0, spare=2, layout="nhd",
                 fill=True):
        g = gen(seed)
        self.lengths, self.page, self.heads, self.dim = lengths, page, heads, dim
        self.new = new if new is not None else [0] * len(lengths)
        pages = [(n + page - 1) // page for n in lengths]
        pool = sum(pages) + spare
        order = torch.randperm(pool, generator=g, device="cuda").tolist()
        indptr, qo = [0], [0]
        for p, n in zip(pages, self.new):
            indptr.append(indptr[-1] + p)
            qo.append(qo[-1] + n)
        self.pages = [order[a:b] for a, b in zip(indptr[:-1], indptr[1:])]
        self.qo = qo
        self.meta = {"qo_indptr_buffer": i32(qo), "paged_kv_indptr_buffer": i32(indptr),
                     "paged_kv_indices_buffer": i32(order),
                     "paged_kv_last_page_len_buffer": i32([(n - 1) % page + 1 if n else 0 for n in lengths])}
        shape, perm = {"nhd": ((pool, page, heads, dim), (0, 1, 2, 3)),
                       "hnd": ((pool, heads, page, dim), (0, 2, 1, 3)),
                       # K and V of a page side by side, rows longer than the head
                       "padded": ((pool, 2, page, heads, dim + 8), None)}[layout]
        if perm:
            self.k = torch.full(shape, float("nan"), dtype=dtype, device="cuda").permute(perm)
            self.v = torch.full(shape, float("nan"), dtype=dtype, device="cuda").permute(perm)
        else:
            both = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
            self.k, self.v = both[:, 0, ..., :dim], both[:, 1, ..., :dim]
        if fill:
            for r, n in enumerate(lengths):
                at = self.where(r, torch.arange(n, device="cuda"))
                self.k[at] = rnd(g, n, heads, dim, dtype=dtype)
                self.v[at] = rnd(g, n, heads, dim, dtype=dtype)
        self.cache = yr.PagedKVCache(self.k, self.v, self.meta)

    def where(self, r, pos):
        pages = torch.tensor(self.pages[r], dtype=torch.long, device="cuda")
        return pages[pos // self.page], pos % self.page


def attention64(q, k, v, scale):
    """(out, lse, sum p |v|, largest sum |q k|) of q [H, D] over k, v [L, Hkv, D] in 64 bits."""
    H, hkv = q.shape[0], k.shape[1]
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    k, v = k.repeat_interleave(H // hkv, 1), v.repeat_interleave(H // hkv, 1)
    s = torch.einsum("hd,lhd->hl", q, k) * scale
    p = torch.softmax(s, 1)
    mass = torch.einsum("hd,lhd->hl", q.abs(), k.abs()).max().item() * abs(scale)
    return torch.einsum("hl,lhd->hd", p, v), torch.logsumexp(s, 1), torch.einsum("hl,lhd->hd", p, v.abs()), mass


def check_attention(out, lse, q, k, v, scale, dtype):
    want, want_lse, pv, mass = attention64(q, k, v, scale)
    ds = 2 * q.shape[-1] * 2 ** -24 * mass
    bound = half_step(dtype) * want.abs() * (1 + 2 ** -6) + pv * (2 * ds + 2 ** -15) + 2 ** -25
    off = (out.to(F64) - want).abs()
    assert (off <= bound).all(), f"out: {(off / bound).max().item():.3g} of the bound"
    if lse is not None:
        off = (lse.to(F64) - want_lse).abs()
        bound = ds + 2 ** -20 * (1 + want_lse.abs())
        assert (off <= bound).all(), f"lse: {(off / bound).max().item():.3g} of the bound"


def run_decode(lengths, *, hq=8, heads=2, dim=128, page=64, dtype=BF16, window=0, scale=None, layout="nhd", seed=0,
               q_scale=2.0):
    b = Batch(lengths, page=page, heads=heads, dim=dim, dtype=dtype, seed=seed, layout=layout)
    q = rnd(gen(seed + 1), len(lengths), hq, dim, dtype=dtype, scale=q_scale)
    out, lse = b.cache.decode(q, return_lse=True, window=window, sm_scale=scale)
    b.cache.check()
    for r, n in enumerate(lengths):
        lo = max(0, n - window) if window else 0
        if n == 0:
            assert (out[r] == 0).all() and (lse[r] == float("-inf")).all()
            continue
        at = b.where(r, torch.arange(lo, n, device="cuda"))
        check_attention(out[r], lse[r], q[r], b.k[at], b.v[at], dim ** -0.5 if scale is None else scale, dtype)
    return b, q, out, lse


# ------------------------------------------------------------------------------------- decode
@pytest.mark.parametrize("page", [1, 3, 16, 40, 64, 256])
def test_decode_lengths_around_pages_and_tiles(page):
    """Lengths of zero and one, at and around the ends of pages and of the kernel's blocks; the
    rest of the last page holds NaN."""
    run_decode([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0], page=page, seed=page)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq,heads", [(1, 1), (4, 4), (8, 1), (12, 4), (16, 1), (34, 2), (40, 8)])
def test_decode_heads_and_types(dtype, dim, hq, heads):
    run_decode([1, 77, 250], hq=hq, heads=heads, dim=dim, dtype=dtype, page=32, seed=hq + dim)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "padded"])
def test_decode_cache_layouts(layout):
    run_decode([33, 200, 5], layout=layout, page=16, seed=3)


@pytest.mark.parametrize("window", [1, 7, 16, 64, 100, 5000])
def test_decode_window(window):
    run_decode([1, 15, 64, 130, 700], window=window, page=16, seed=window)


def test_decode_scale_and_peaked_weights():
    run_decode([300, 20], scale=0.5, seed=5)
    run_decode([300, 20], scale=-0.1, seed=6)
    run_decode([300, 20], scale=0.0, seed=7)
    run_decode([900, 33], q_scale=30.0, seed=8)              # nearly all weight on one position
    run_decode([900, 33], q_scale=30.0, seed=8, dtype=F16)


@pytest.mark.parametrize("hq,heads,lengths", [(8, 1, [40000]), (8, 2, [20011, 3, 0, 9000]), (32, 8, [4097] * 3),
                                              (16, 1, [17777, 60])])
def test_decode_split_over_long_lengths(hq, heads, lengths):
    b, q, out, lse = run_decode(lengths, hq=hq, heads=heads, seed=11)
    again = b.cache.decode(q, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)     # no order of arrival in it


@pytest.mark.parametrize("page", [1, 2, 7, 16, 48])
@pytest.mark.parametrize("window", [0, 1500])
def test_decode_lengths_of_many_short_pages(page, window):
    """Requests of hundreds of pages beside short ones, from ranges that begin inside them."""
    run_decode([2500, 1, 650, 0, 1037], page=page, window=window, seed=20 + page)
    run_decode([700], hq=8, heads=1, dim=256, page=page, window=window, seed=40 + page)


def test_decode_many_short_requests_beside_long_ones():
    """Where the work is cut, the end of every request counts: cuts fall behind the last block of
    one and inside others."""
    lengths = [(53 * i) % 420 + (6000 if i in (11, 12, 40) else 0) for i in range(48)]
    run_decode(lengths, hq=4, heads=4, dim=64, page=16, seed=50)
    run_decode(lengths[::-1], hq=16, heads=2, dim=128, page=64, seed=51, dtype=F16)
    run_decode([270] * 37 + [0, 4000], hq=2, heads=1, dim=128, page=16, seed=52)


@pytest.mark.parametrize("hq,heads,dim,page,window", [(4, 4, 128, 16, 0), (32, 4, 128, 64, 0), (64, 4, 128, 7, 0),
                                                      (8, 4, 256, 48, 0), (64, 4, 64, 16, 0), (80, 4, 64, 64, 0),
                                                      (16, 4, 128, 16, 50), (16, 4, 64, 1, 2000)])
def test_decode_many_short_requests_warp_by_warp(hq, heads, dim, page, window):
    """Hundreds of short (request, head)s, a few long ones among them that run through many warps
    and CTAs: at the start, in the middle, next to one another and at the end."""
    lengths = [(29 * i) % 131 for i in range(165)]
    for at, n in ((0, 5000), (80, 2100), (81, 700), (82, 3300), (164, 1500)):
        lengths[at] = n
    dtype = F16 if hq == 32 else BF16
    b, q, out, lse = run_decode(lengths, hq=hq, heads=heads, dim=dim, page=page, window=window, dtype=dtype, seed=70)
    again = b.cache.decode(q, return_lse=True, window=window)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    run_decode([1] * 400 + [0] * 7 + [17, 16, 15], hq=hq, heads=heads, dim=dim, page=page, window=window, seed=71)
    run_decode([512] * 170, hq=hq, heads=heads, dim=dim, page=max(page, 7), window=window, seed=72)


@pytest.mark.parametrize("lengths,heads,hurt,entry", [([100] * 190, 4, 77, 3), ([3000, 60, 3100], 2, 2, 150),
                                                      ([40] * 300 + [2000], 4, 300, 60)])
def test_decode_bad_pages_in_either_form(lengths, heads, hurt, entry):
    """A broken page number, in a batch of many short requests or far into a long one: its request
    loses those positions, the others keep their bits; an emptied request is zeros."""
    b = Batch(lengths, heads=heads, page=16, seed=80)
    q = rnd(gen(81), len(lengths), 4 * heads, 128)
    good = b.cache.decode(q)
    b.cache.check()
    idx, ptr = b.meta["paged_kv_indices_buffer"], b.meta["paged_kv_indptr_buffer"]
    keep, at = idx.clone(), int(ptr[hurt]) + entry
    for bad in (-1, b.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        idx.copy_(keep)
        idx[at] = bad
        out = b.cache.decode(q)
        with pytest.raises(N.YpkError, match="outside the pool"):
            b.cache.check()
        others = [r for r in range(len(lengths)) if r != hurt]
        assert torch.equal(out[others], good[others])
        pos = torch.arange(lengths[hurt], device="cuda")
        where = b.where(hurt, pos[(pos < 16 * entry) | (pos >= 16 * (entry + 1))])
        check_attention(out[hurt], None, q[hurt], b.k[where], b.v[where], 128 ** -0.5, BF16)
    idx.copy_(keep)
    b.meta["paged_kv_last_page_len_buffer"][hurt] = 17          # longer than a page
    out, lse = b.cache.decode(q, return_lse=True)
    with pytest.raises(N.YpkError, match="out of order"):
        b.cache.check()
    assert (out[hurt] == 0).all() and (lse[hurt] == float("-inf")).all()
    for r in (0, len(lengths) // 2):
        if r != hurt:
            where = b.where(r, torch.arange(lengths[r], device="cuda"))
            check_attention(out[r], lse[r], q[r], b.k[where], b.v[where], 128 ** -0.5, BF16)


def test_decode_nan_in_a_seen_position_shows():
    """A NaN among the seen K rows makes the heads that read it NaN, and no others."""
    for n, at in ((100, 17), (5000, 4999), (1, 0)):
        b = Batch([n, 50], seed=30)
        b.k[b.where(0, torch.tensor([at], device="cuda"))[0], at % 64, 1, 5] = float("nan")
        q = rnd(gen(31), 2, 8, 128)
        out, lse = b.cache.decode(q, return_lse=True)
        assert torch.isnan(out[0, 4:]).all() and torch.isnan(lse[0, 4:]).all()
        assert torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all()


def test_decode_many_requests():
    lengths = [(37 * i) % 190 for i in range(700)]
    run_decode(lengths, hq=4, heads=1, dim=64, page=16, seed=12)
    # as many as a call takes: the tables cost the ring a block per warp
    lengths = [(7 * i) % 50 for i in range(4096)]
    b = Batch(lengths, heads=1, dim=128, page=16, seed=13)
    q = rnd(gen(14), 4096, 16, 128)
    out = b.cache.decode(q)
    b.cache.check()
    for r in range(0, 4096, 97):
        at = b.where(r, torch.arange(lengths[r], device="cuda"))
        if lengths[r]:
            check_attention(out[r], None, q[r], b.k[at], b.v[at], 128 ** -0.5, BF16)
        else:
            assert (out[r] == 0).all()


def test_decode_query_views_outputs_and_rows_behind():
    """q as the packed rows of a fused projection; fewer rows than requests; out given, its rows
    behind the last sequence as they were."""
    b = Batch([50, 80, 20], heads=2, seed=13)
    rows = rnd(gen(14), 3, 2, 4 + 2, 128)
    buf = torch.full((5, 2, 4, 128), 7.0, dtype=BF16, device="cuda")
    out = b.cache.decode(rows[:2, :, :4], out=buf[:2])
    assert out.data_ptr() == buf.data_ptr() and (buf[2:] == 7).all()
    for r in range(2):
        at = b.where(r, torch.arange(b.lengths[r], device="cuda"))
        check_attention(out[r].reshape(8, 128), None, rows[r, :, :4].reshape(8, 128), b.k[at], b.v[at], 128 ** -0.5, BF16)
    # the empty call
    assert b.cache.decode(rows[:0, :, :4]).shape == (0, 2, 4, 128)


def test_decode_bad_tables_are_reported_and_left_out():
    """Broken entries (walked on the CPU in test_serving_cpu.py) never become addresses."""
    b = Batch([100, 100, 100], page=16, seed=15)
    q = rnd(gen(16), 3, 8, 128)
    good = b.cache.decode(q)
    b.cache.check()
    idx, ptr = b.meta["paged_kv_indices_buffer"], b.meta["paged_kv_indptr_buffer"]
    keep = idx.clone()
    for bad in (-1, b.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        idx.copy_(keep)
        idx[2] = bad                                     # request 0 loses positions 32..47
        out = b.cache.decode(q)
        with pytest.raises(N.YpkError, match="outside the pool"):
            b.cache.check()
        assert torch.equal(out[1:], good[1:])
        pos = torch.cat((torch.arange(32, device="cuda"), torch.arange(48, 100, device="cuda")))
        at = b.where(0, pos)
        check_attention(out[0], None, q[0], b.k[at], b.v[at], 128 ** -0.5, BF16)
    idx.copy_(keep)
    keep_ptr = ptr.clone()
    # (entry, value, requests whose run is broken, requests whose run is as it was); a run that
    # stays inside the page list is a run, if not the one that was meant: its result is not looked at
    for at, bad, empty, same in ((1, -3, (0, 1), (2,)), (1, 10 ** 6, (0, 1), (2,)), (3, 2 ** 31 - 1, (2,), (0, 1)),
                                 (2, 0, (1,), (0,))):
        ptr.copy_(keep_ptr)
        ptr[at] = bad
        out, lse = b.cache.decode(q, return_lse=True)
        with pytest.raises(N.YpkError, match="out of order"):
            b.cache.check()
        for r in empty:
            assert (out[r] == 0).all() and (lse[r] == float("-inf")).all()
        for r in same:
            assert torch.equal(out[r], good[r])
    ptr.copy_(keep_ptr)
    b.meta["paged_kv_last_page_len_buffer"][0] = 17      # more than a page
    out, lse = b.cache.decode(q, return_lse=True)
    with pytest.raises(N.YpkError, match="out of order"):
        b.cache.check()
    assert (out[0] == 0).all() and torch.equal(out[1:], good[1:])


def test_decode_offsets_past_32_bits():
    """A pool whose rows lie beyond 2^32 elements: 4300 pages of 4 MB per cache."""
    page, heads = 4096, 4
    pool = (1 << 32) // (page * heads * 128) + 5
    k = torch.empty(pool, page, heads, 128, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    g = gen(17)
    far = [pool - 1, 0, pool - 2]
    for p in far:
        k[p], v[p] = rnd(g, page, heads, 128), rnd(g, page, heads, 128)
    meta = {"qo_indptr_buffer": i32([0, 1]), "paged_kv_indptr_buffer": i32([0, 3]), "paged_kv_indices_buffer": i32(far),
            "paged_kv_last_page_len_buffer": i32([100])}
    c = yr.PagedKVCache(k, v, meta)
    q, kn, vn = rnd(g, 1, 8, 128), rnd(g, 1, heads, 128), rnd(g, 1, heads, 128)
    c.append(kn, vn)
    assert torch.equal(k[pool - 2, 99], kn[0]) and torch.equal(v[pool - 2, 99], vn[0])
    out = c.decode(q)
    c.check()
    kk = torch.cat((k[far[0]], k[far[1]], k[far[2], :100]))
    vv = torch.cat((v[far[0]], v[far[1]], v[far[2], :100]))
    check_attention(out[0], None, q[0], kk, vv, 128 ** -0.5, BF16)


# ------------------------------------------------------------------------------------- append
def tables(positions, rot, dtype, theta=500000.0):
    f = theta ** (-torch.arange(0, rot, 2, dtype=F64, device="cuda") / rot)
    a = torch.arange(positions, dtype=F64, device="cuda")[:, None] * f
    a = torch.cat((a, a), 1)
    return a.cos().to(dtype), a.sin().to(dtype)


def rotated64(x, w, eps, cos, sin):
    """(y, |a c| + |b s|) of rows x [n, heads, D] in 64 bits; cos, sin [n, rot] or None."""
    x = x.to(F64)
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.to(F64)
    if cos is None:
        return x, x.abs()
    rot = cos.shape[1]
    h = rot // 2
    c, s = cos.to(F64)[:, None], sin.to(F64)[:, None]
    a, b, rest = x[..., :h], x[..., h:rot], x[..., rot:]
    y = torch.cat((a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:], rest), -1)
    size = torch.cat(((a * c[..., :h]).abs() + (b * s[..., :h]).abs(), (b * c[..., h:]).abs() + (a * s[..., h:]).abs(),
                      rest.abs()), -1)
    return y, size


def run_append(lengths, new, *, hq=8, heads=2, dim=128, page=16, dtype=BF16, table=None, rot=None, norm=False,
               packed=True, pad=0, layout="nhd", seed=0, with_q=True, rotate=True):
    b = Batch(lengths, new, page=page, heads=heads, dim=dim, dtype=dtype, seed=seed, layout=layout)
    g, n = gen(seed + 100), sum(new) + pad
    G = hq // heads
    if packed:
        rows = rnd(g, n, heads, G + 2, dim, dtype=dtype)
        q, k, v = rows[:, :, :G], rows[:, :, G], rows[:, :, G + 1]
    else:
        q, k, v = rnd(g, n, hq, dim, dtype=dtype), rnd(g, n, heads, dim, dtype=dtype), rnd(g, n, heads, dim, dtype=dtype)
    cos = sin = None
    if rotate:
        cos, sin = tables(max(lengths), rot or dim, table or dtype)
    qw = kw = None
    if norm:
        qw, kw = rnd(g, dim, dtype=dtype) * 0.2 + 1, rnd(g, dim, dtype=dtype) * 0.2 + 1
    want_k, want_v = b.k.clone(), b.v.clone()
    out = torch.full((n, hq, dim), 9.0, dtype=dtype, device="cuda") if with_q else None
    got = b.cache.append(k, v, q=q if with_q else None, q_out=out, cos=cos, sin=sin, q_norm=qw if with_q else None,
                         k_norm=kw, eps=1e-5)
    b.cache.check()
    rel = (dim / 2 + 8) * 2 ** -24 if norm else 3 * 2 ** -24
    tiny = 2 ** -25 if dtype == F16 else 0.0          # half of fp16's smallest step

    def near(x, y, size, what):
        off = (x.to(F64) - y).abs()
        bound = half_step(dtype) * (1 + 2 ** -6) * y.abs() + 2 * rel * size + tiny
        assert (off <= bound).all(), f"{what}: {(off - bound).max().item():.3g} past the bound"

    for r, (length, m) in enumerate(zip(lengths, new)):
        rows_r = slice(b.qo[r], b.qo[r + 1])
        pos = torch.arange(length - m, length, device="cuda")
        at = b.where(r, pos)
        c, s = (cos[pos], sin[pos]) if rotate else (None, None)
        y, size = rotated64(k[rows_r], kw, 1e-5, c, s)
        near(b.k[at], y, size, f"K of request {r}")
        assert torch.equal(b.v[at], v[rows_r])
        want_k[at], want_v[at] = b.k[at], v[rows_r]
        if with_q:
            y, size = rotated64(q[rows_r].reshape(m, hq, dim), qw, 1e-5, c, s)
            near(got[rows_r], y, size, f"q of request {r}")
    # nothing else was written: bits, since the rest of the pool holds NaN
    assert torch.equal(b.k.contiguous().view(torch.int16), want_k.contiguous().view(torch.int16))
    assert torch.equal(b.v.contiguous().view(torch.int16), want_v.contiguous().view(torch.int16))
    if with_q:
        assert (got[sum(new):] == 9).all()
    else:
        assert got is None
    return b


@pytest.mark.parametrize("page", [1, 3, 16, 64])
def test_append_lengths_and_padding(page):
    run_append([1, 5, 64, 65, 200, 0, 17], [1, 5, 1, 3, 199, 0, 0], page=page, pad=3, seed=page)


@pytest.mark.parametrize("dtype,table", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 16), (128, 128), (128, 64), (256, 256), (256, 32)])
def test_append_types_and_rotated_parts(dtype, table, dim, rot):
    run_append([40, 3, 111], [7, 3, 1], dim=dim, rot=rot, dtype=dtype, table=table, seed=dim + rot)
    run_append([40, 3, 111], [7, 3, 1], dim=dim, rot=rot, dtype=dtype, table=table, norm=True, packed=False, seed=dim)


@pytest.mark.parametrize("hq,heads", [(1, 1), (5, 1), (7, 7), (12, 4), (64, 8)])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "padded"])
def test_append_heads_and_layouts(hq, heads, layout):
    run_append([33, 70], [33, 2], hq=hq, heads=heads, layout=layout, seed=hq)


def test_append_without_queries_rotation_or_norm():
    run_append([50, 9], [20, 9], with_q=False, seed=1)
    run_append([50, 9], [20, 9], rotate=False, seed=2)
    run_append([50, 9], [20, 9], rotate=False, norm=True, with_q=False, seed=3)


def test_append_many_requests_and_long_prompts():
    run_append([(13 * i) % 90 + 1 for i in range(500)], [1] * 500, hq=4, heads=1, dim=64, page=16, seed=4)
    run_append([3000, 1111], [3000, 1000], hq=8, heads=2, page=64, seed=5)


def test_append_in_place_queries():
    b = Batch([30, 7], [10, 7], seed=6)
    g = gen(7)
    k, v, q = rnd(g, 17, 2, 128), rnd(g, 17, 2, 128), rnd(g, 17, 8, 128)
    cos, sin = tables(64, 128, BF16)
    w = rnd(g, 128) * 0.1 + 1
    apart = b.cache.append(k, v, q=q, cos=cos, sin=sin, q_norm=w)
    same = b.cache.append(k, v, q=q, q_out=q, cos=cos, sin=sin, q_norm=w)
    assert same.data_ptr() == q.data_ptr() and torch.equal(same, apart)


def test_append_equals_the_attention_task_bit_for_bit():
    """K and V rows appended here are those the graph's attention task appends."""
    from tests.util import onepass_kernel
    R, hq, hkv, D = 3, 8, 2, 128
    lengths = [65, 1, 130]
    b = Batch(lengths, [1] * R, seed=8)
    b.k.nan_to_num_(0.5)
    b.v.nan_to_num_(0.5)
    qkv = rnd(gen(9), 8, hkv * 6 * D)
    cos, sin = O.rope_tables(D, 500000.0, 256)
    cos, sin = cos.cuda(), sin.cuda()
    kc, vc = b.k.clone(), b.v.clone()
    ypk = onepass_kernel(8, b.meta, max_requests=R, max_pages=kc.shape[0], page_size=64, max_seq_length=256)
    out = torch.zeros(8, hq * D, dtype=BF16, device="cuda")
    ypk.paged_attention_layer(ypk.attach_input(qkv, "qkv"), ypk.attach_input(kc, "kc"), ypk.attach_input(vc, "vc"),
                              None, None, ypk.attach_input(cos, "cos"), ypk.attach_input(sin, "sin"),
                              ypk.attach_input(out, "out"), (R, hkv, 1), (128, 1, 1))
    ypk.compile()
    ypk(batch=R)
    rows = qkv.view(8, hkv, 6, D)[:R]
    q = b.cache.append(rows[:, :, 4], rows[:, :, 5], q=rows[:, :, :4], cos=cos, sin=sin)
    assert torch.equal(b.k, kc) and torch.equal(b.v, vc)
    got = b.cache.decode(q).view(R, hq * D)
    b.cache.check()
    # two ways to the same attention, each within a rounding and its weights' 16-bit rounding
    assert (got.float() - out[:R].float()).abs().max() <= 2e-2
    ypk.finalize()


def test_append_bad_tables_are_reported_and_dropped():
    b = Batch([40, 40], [2, 2], page=16, seed=10)
    g = gen(11)
    k, v, q = rnd(g, 4, 2, 128), rnd(g, 4, 2, 128), rnd(g, 4, 8, 128)
    cos, sin = tables(40, 128, BF16)
    before = b.k.clone(), b.v.clone()

    def run(text, kept, **kw):
        """Rows `kept` of the call arrive, the others leave everything as it was."""
        b.k.copy_(before[0])
        b.v.copy_(before[1])
        out = torch.full((4, 8, 128), 9.0, dtype=BF16, device="cuda")
        b.cache.append(k, v, q=q, q_out=out, **dict(dict(cos=cos, sin=sin), **kw))
        with pytest.raises(N.YpkError, match=text):
            b.cache.check()
        for row in range(4):
            assert (out[row] == 9).all().item() == (row not in kept)
        changed = (b.v.view(torch.int16) != before[1].view(torch.int16)).any(-1).any(-1)
        assert int(changed.sum()) == len(kept)

    b.meta["paged_kv_indices_buffer"][2] = 10 ** 6
    run("outside the pool", (2, 3))
    b.meta["paged_kv_indices_buffer"][2] = b.pages[0][2]
    run("outside the rotary tables", (0, 2), cos=cos[:39], sin=sin[:39])
    b.meta["paged_kv_last_page_len_buffer"][1] = 17
    run("out of order", (0, 1))
    b.meta["paged_kv_last_page_len_buffer"][1] = 8
    b.meta["qo_indptr_buffer"].copy_(i32([0, 0, 4]))      # request 1 brings four, request 0 none
    b.meta["paged_kv_indptr_buffer"].copy_(i32([0, 5, 6]))
    b.meta["paged_kv_last_page_len_buffer"][1] = 3        # ... but is three tokens long
    run("more new tokens", (1, 2, 3))


# ----------------------------------------------------------------------------------- logprobs
def order_keys(x):
    bits = (x.float() + 0.0).view(torch.int32).long()
    return torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))


def check_logprobs(logits, tokens, top_k, vocab=None):
    vocab = logits.shape[1] if vocab is None else vocab
    got = yr.token_logprobs(logits, tokens, top_k=top_k, valid_cols=vocab)
    x = logits[:, :vocab].to(F64)
    t = tokens.view(-1)
    top = x.max(1, keepdim=True).values
    empty = top == float("-inf")
    z = torch.where(empty, 0.0, x - torch.where(empty, 0.0, top))
    w = torch.where(x == float("-inf"), 0.0, z.exp())
    total = w.sum(1, keepdim=True)
    logp = torch.where(x == float("-inf"), float("-inf"), z - total.log())
    inside = (t >= 0) & (t < vocab)
    want = torch.where(inside, logp.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0], float("-inf"))

    def near(a, b, what):
        a = a.to(F64)
        assert torch.equal(a == float("-inf"), b == float("-inf")), what
        fine = torch.isfinite(b)
        assert torch.isfinite(a[fine]).all(), what
        off = (a[fine] - b[fine]).abs() - (2 ** -15 + 2 * 2 ** -24 * b[fine].abs())
        assert not off.numel() or off.max() <= 0, f"{what}: {off.max().item():.3g} past the bound"

    near(got.logprob, want, "logprob")
    entropy = -torch.where(w > 0, w * torch.where(w > 0, logp, 0.0), 0.0).sum(1) / total[:, 0].clamp(min=1e-300)
    entropy = torch.where(empty[:, 0], 0.0, entropy)
    off = (got.entropy.to(F64) - entropy).abs()
    assert (off <= 2 ** -14 * (1 + entropy)).all(), f"entropy: off by {off.max().item():.3g}"
    if top_k:
        at = torch.topk(order_keys(logits[:, :vocab]) * (1 << 20) - torch.arange(vocab, device="cuda"), top_k, 1).indices
        assert torch.equal(got.top_token, at), "top tokens"
        near(got.top_logprob, logp.gather(1, at), "top_logprob")
    else:
        assert got.top_logprob is None and got.top_token is None
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 31, 255, 1000, 4097, 32003, 128256])
def test_logprobs_sizes_and_types(dtype, vocab):
    g = gen(vocab)
    for rows in (1, 5):
        x = rnd(g, rows, vocab, dtype=dtype, scale=3.0)
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        for k in (0, 1, 5, 32):
            check_logprobs(x, t, min(k, vocab))


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 37, 150, 700])
def test_logprobs_rows(rows):
    g = gen(rows)
    x = rnd(g, rows, 20011, scale=3.0)
    t = torch.randint(0, 20011, (rows, 1), generator=g, device="cuda")
    check_logprobs(x, t, 20)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_logprobs_padding_strides_and_alignment(dtype):
    """Columns behind the vocabulary hold NaN and infinities; rows start at any element."""
    g = gen(1)
    for first in (0, 1, 2, 3, 5, 7):
        for pad in (0, 1, 6, 13):
            store = torch.full((6, 1500 + first + pad), float("nan"), dtype=dtype, device="cuda")
            store[:, -1:] = float("inf")
            x = store[:, first:]
            x[:, :1490] = rnd(g, 6, 1490, dtype=dtype, scale=2.0)
            check_logprobs(x, torch.randint(0, 1490, (6,), generator=g, device="cuda"), 9, vocab=1490)
            check_logprobs(x[::2], torch.randint(0, 1490, (3,), generator=g, device="cuda"), 9, vocab=1490)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_logprobs_ties_go_to_the_lower_column(dtype):
    x = torch.zeros(4, 9000, dtype=dtype, device="cuda")
    x[1, 5000:] = 1.0
    x[2] = (torch.arange(9000, device="cuda") % 3).to(dtype)
    x[3, ::2] = -0.0                                       # the same value as 0.0
    got = check_logprobs(x, torch.tensor([0, 1, 2, 3], device="cuda"), 32)
    assert got.top_token[0].tolist() == list(range(32)) and got.top_token[3].tolist() == list(range(32))


@pytest.mark.parametrize("rising", [True, False])
def test_logprobs_sorted_rows(rising):
    """Every column beats all before it, or none does."""
    for n, rows in ((300, 2), (40000, 2), (5000, 200)):
        x = torch.linspace(-5, 5, n, device="cuda").expand(rows, n).contiguous()
        x = x if rising else x.flip(1)
        check_logprobs(x, torch.full((rows,), n // 2, device="cuda"), 32)
        check_logprobs(x.to(BF16), torch.full((rows,), n // 2, device="cuda"), 7)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 700])
def test_logprobs_high_columns_crowded(dtype, rows):
    """Thousands of high values in the columns of a few threads, equal or not: more than the list of
    candidates holds."""
    g = gen(8)
    n, width = 60000, 8 if dtype == BF16 else 4
    col = torch.arange(n, device="cuda")
    for block in (512, 64):
        crowd = ((col // width) % block) % 24 == 5
        x = rnd(g, rows, n, dtype=dtype)
        t = torch.randint(0, n, (rows,), generator=g, device="cuda")
        check_logprobs(torch.where(crowd, x + 9, x), t, 32)
        check_logprobs(torch.where(crowd, torch.full_like(x, 9), x), t, 32)
        few = torch.where(col % 9001 == 77, x + 20, torch.full_like(x, float("-inf")))
        check_logprobs(few, t, 20)                  # fewer columns than alternatives


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_logprobs_masked_rows(dtype):
    g = gen(3)
    ninf, low = float("-inf"), torch.finfo(dtype).min
    x = rnd(g, 9, 4000, dtype=dtype, scale=2.0)
    x[0] = ninf                                            # nothing is left
    x[1, 1:] = ninf                                        # one column is
    x[2, :3990] = ninf
    x[3, torch.rand(4000, generator=g, device="cuda") < 0.9] = ninf
    x[4] = low                                             # a mask of the lowest value everywhere: uniform
    x[5, 10:] = low
    x[6, 10:] = low
    x[6, 20:] = ninf
    x[7] = torch.finfo(dtype).max
    x[8, :5] = torch.finfo(dtype).max
    got = check_logprobs(x, torch.tensor([0, 0, 3999, 7, 4, 3, 15, 9, 2], device="cuda"), 12)
    # one column: ln 2 (log2 2^e - e), e the rounding of the reference, both functions within 2 ulp
    # of a number next to 1: 2^-21
    assert got.entropy[0] == 0 and 0 <= got.entropy[1] <= 2 ** -21 and (got.top_logprob[0] == ninf).all()
    assert got.top_token[0].tolist() == list(range(12))
    assert abs(got.entropy[4].item() - math.log(4000)) < 1e-3


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [1, 150])
def test_logprobs_far_values(dtype, rows):
    """Rows at every distance from zero: values and masks around the borders of the exponent's range.
    A weight is then off by 2^-24 of the reference's size more, as y = x log2 e - r is: far rows
    get that on top of the bound, which check_logprobs takes for values of ordinary size."""
    g = gen(40)
    big = torch.finfo(dtype).max
    for base in (0.0, 100.0, 6e4, 1e6, 1e9, 2.0 ** 30, 2.0 ** 31, 1e10, 1e30, 2.3e38, 3.3e38):
        for sign in (1, -1):
            if base > big:
                continue
            x = (torch.randn(rows, 9000, generator=g, device="cuda") + sign * base).clamp(-big, big).to(dtype)
            x[:, 7000:] = -big
            x[:, 8000:] = float("-inf")
            t = torch.randint(0, 9000, (rows,), generator=g, device="cuda")
            got = yr.token_logprobs(x, t, top_k=3)
            want = torch.log_softmax(x.to(F64), 1)
            p = want.exp()
            entropy = -torch.where(p > 0, p * want, 0.0).sum(1)
            off = 2 ** -14 * (1 + entropy) + 2 ** -22 * min(base, 2.0 ** 30) * 2 ** -7
            assert ((got.entropy.to(F64) - entropy).abs() <= off).all(), (base, sign)
            lp, w = got.logprob.to(F64), want.gather(1, t[:, None])[:, 0]
            w = torch.where(torch.isinf(w.to(F32)), float("-inf"), w)        # more than fp32 holds
            seen = w > float("-inf")
            assert torch.equal(lp > float("-inf"), seen)
            assert ((lp - w).abs()[seen] <= (2 ** -15 + 2 ** -22 * min(base, 2.0 ** 30) * 2 ** -7 + 2 ** -22 * w.abs())[seen]).all()
            at = torch.topk(order_keys(x) * (1 << 20) - torch.arange(9000, device="cuda"), 3, 1).indices
            assert torch.equal(got.top_token, at)


@pytest.mark.parametrize("rows", [1, 200])
def test_logprobs_nan_and_infinite_rows(rows):
    g = gen(4)
    x = rnd(g, rows + 2, 5000, scale=2.0)
    clean = x.clone()
    x[0, 1234], x[1, 77] = float("nan"), float("inf")
    t = torch.zeros(rows + 2, dtype=torch.int64, device="cuda")
    got = yr.token_logprobs(x, t, top_k=3)
    for a in (got.logprob, got.entropy, got.top_logprob[:, 0]):
        assert torch.isnan(a[:2]).all() and torch.isfinite(a[2:]).all()
    assert got.top_token[1, 0] == 77 and 1234 not in got.top_token[0].tolist()
    assert torch.equal(got.top_token[2:], yr.token_logprobs(clean, t, top_k=3).top_token[2:])


def test_logprobs_tokens_outside_the_vocabulary():
    x = rnd(gen(5), 5, 100)
    t = torch.tensor([-1, 100, 99, -2 ** 63, 2 ** 63 - 1], device="cuda")
    check_logprobs(x, t, 3)
    check_logprobs(x, torch.tensor([60, 50, 49, 0, 1], device="cuda"), 3, vocab=50)


def test_logprobs_offsets_past_32_bits():
    """The last rows start beyond 2^32 elements."""
    ld = 200000
    rows = (1 << 32) // ld + 3
    store = torch.empty(rows, ld, dtype=BF16, device="cuda")
    x = store[:, :1000]
    g = gen(6)
    far = slice(rows - 4, rows)
    x.zero_()
    x[far] = rnd(g, 4, 1000, scale=2.0)
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    t[far] = torch.tensor([5, 6, 7, 999], device="cuda")
    got = yr.token_logprobs(x, t, top_k=4)
    near = yr.token_logprobs(x[far].contiguous(), t[far].contiguous(), top_k=4)
    for a, b in zip(got, near):
        assert torch.equal(a[far], b)


# ------------------------------------------------------------------------------------ together
def decode_loop(b, cos, sin, k_all, v_all, q_all, steps, graph=None):
    """`steps` decode steps over batch b: tables advance by one token, append, attend."""
    outs = []
    for i in range(steps):
        for r in range(len(b.lengths)):
            b.lengths[r] += 1
        pages = [(n + b.page - 1) // b.page for n in b.lengths]
        indptr = [0]
        flat = []
        for r, p in enumerate(pages):
            flat += b.pages[r][:p]
            indptr.append(len(flat))
        b.meta["paged_kv_indptr_buffer"].copy_(i32(indptr))
        b.meta["paged_kv_indices_buffer"][:len(flat)].copy_(i32(flat))
        b.meta["paged_kv_last_page_len_buffer"].copy_(i32([(n - 1) % b.page + 1 for n in b.lengths]))
        if graph is not None:
            graph["k"].copy_(k_all[i])
            graph["v"].copy_(v_all[i])
            graph["q"].copy_(q_all[i])
            graph["graph"].replay()
            outs.append(graph["out"].clone())
        else:
            q = b.cache.append(k_all[i], v_all[i], q=q_all[i], cos=cos, sin=sin)
            outs.append(b.cache.decode(q))
    b.cache.check()
    return outs


def make_steps(seed, R=3, steps=20):
    g = gen(seed)
    b = Batch([40, 1, 100], [1] * R, page=16, heads=2, seed=seed, spare=8)
    spare = [p for p in range(b.k.shape[0]) if all(p not in x for x in b.pages)]
    for r in range(R):
        b.pages[r] = b.pages[r] + [spare.pop(), spare.pop()]
    b.k.nan_to_num_(0.25)
    b.v.nan_to_num_(0.25)
    return (b, [rnd(g, R, 2, 128) for _ in range(steps)], [rnd(g, R, 2, 128) for _ in range(steps)],
            [rnd(g, R, 8, 128, scale=2.0) for _ in range(steps)])


def test_append_and_decode_together_eager_and_captured():
    """Twenty decode steps of three requests that grow over page ends, against attention over the
    whole rotated history; then the same steps as replays of one captured graph: the tables'
    contents change between replays, the results are the same bits."""
    steps = 20
    cos, sin = tables(256, 128, BF16)
    b, ks, vs, qs = make_steps(20, steps=steps)
    start = list(b.lengths)
    outs = decode_loop(b, cos, sin, ks, vs, qs, steps)
    for r in range(3):
        at = b.where(r, torch.arange(b.lengths[r], device="cuda"))
        hist_k, hist_v = b.k[at], b.v[at]
        for i in range(steps):
            n = start[r] + i + 1
            y, _ = rotated64(ks[i][r:r + 1], None, 0, cos[n - 1:n], sin[n - 1:n])
            assert torch.equal(hist_k[n - 1].to(F64), y[0].to(BF16).to(F64)) or \
                (hist_k[n - 1].to(F64) - y[0]).abs().max() <= 2 ** -8 * 4
            q, _ = rotated64(qs[i][r:r + 1], None, 0, cos[n - 1:n], sin[n - 1:n])
            want, _, pv, mass = attention64(q[0].to(BF16), hist_k[:n], hist_v[:n], 128 ** -0.5)
            # the rotated query is a rounding away from the kernel's where fp32 and 64 bits fall on
            # different sides: half a step on each score term
            ds = (2 ** -8 + 2 * 128 * 2 ** -24) * mass
            assert ((outs[i][r].to(F64) - want).abs() <= 2 ** -8 * want.abs() + pv * 2 * ds).all()
    b2, ks2, vs2, qs2 = make_steps(20, steps=steps)
    graph = {"k": ks2[0].clone(), "v": vs2[0].clone(), "q": qs2[0].clone()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                     # warm-up off the capture
        b2.cache.decode(graph["q"])
    torch.cuda.current_stream().wait_stream(side)
    graph["graph"] = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph["graph"]):
        q = b2.cache.append(graph["k"], graph["v"], q=graph["q"], cos=cos, sin=sin)
        graph["out"] = b2.cache.decode(q)
    for a, c in zip(outs, decode_loop(b2, cos, sin, ks2, vs2, qs2, steps, graph)):
        assert torch.equal(a, c)


def test_two_streams_and_two_graphs_at_once():
    """Calls on two streams, and two captured graphs that replay at the same time, share nothing."""
    a, b = Batch([9000, 20], seed=21), Batch([7000, 4000], seed=22)
    qa, qb = rnd(gen(23), 2, 8, 128), rnd(gen(24), 2, 8, 128)
    x, y = rnd(gen(25), 3, 128256), rnd(gen(26), 3, 128256)
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    want = a.cache.decode(qa), b.cache.decode(qb), yr.token_logprobs(x, t, top_k=5), yr.token_logprobs(y, t, top_k=5)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(50):
        with torch.cuda.stream(s1):
            got.append((0, a.cache.decode(qa)))
            got.append((2, yr.token_logprobs(x, t, top_k=5)))
        with torch.cuda.stream(s2):
            got.append((1, b.cache.decode(qb)))
            got.append((3, yr.token_logprobs(y, t, top_k=5)))
    torch.cuda.synchronize()

    def same(i, out):
        return torch.equal(out, want[i]) if i < 2 else all(torch.equal(p, q) for p, q in zip(out, want[i]))

    assert all(same(i, out) for i, out in got)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1, l1 = a.cache.decode(qa), yr.token_logprobs(x, t, top_k=5)
    with torch.cuda.graph(g2):
        o2, l2 = b.cache.decode(qb), yr.token_logprobs(y, t, top_k=5)
    for _ in range(50):
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
    torch.cuda.synchronize()
    assert same(0, o1) and same(1, o2) and same(2, l1) and same(3, l2)


def test_logprobs_results_stand_by_themselves():
    """The four results are ordinary contiguous tensors apart from one another, whatever else is done
    with them."""
    x, k = rnd(gen(90), 5, 1000), torch.arange(5, device="cuda")
    keep = [t.clone() for t in yr.token_logprobs(x, k, top_k=3)]
    for i in range(4):
        p = yr.token_logprobs(x, k, top_k=3)
        assert [tuple(t.shape) for t in p] == [(5,), (5,), (5, 3), (5, 3)]
        assert [t.dtype for t in p] == [F32, F32, F32, torch.int64] and all(t.is_contiguous() for t in p)
        p[i].zero_()
        for j in range(4):
            assert torch.equal(p[j], keep[j] * 0 if i == j else keep[j]), (i, j)
        copy = p.top_token.to("cpu")
        del p
        torch.empty(4096, device="cuda").fill_(7)
        assert i == 3 or torch.equal(copy, keep[3].cpu())
    with pytest.raises(N.YpkError, match="top_k"):
        yr.token_logprobs(x, k, top_k=2 ** 31 - 1)


def test_calls_wait_for_what_runs_before_them():
    """Inputs written just before the call by a long kernel, a copy or a fill on the same stream, or on
    another one behind an event; outputs read right behind it."""
    b = Batch([700, 90], [1, 1], page=64, seed=60)
    g = gen(61)
    q, n = rnd(g, 2, 8, 128), rnd(g, 2, 2, 128)
    x, t = rnd(g, 2, 50000), torch.tensor([3, 4], device="cuda")
    cos, sin = tables(1024, 128, BF16)
    rotated = b.cache.append(n, n, q=q, cos=cos, sin=sin).clone()
    want, lp = b.cache.decode(rotated).clone(), yr.token_logprobs(x, t, top_k=4)
    side, slow = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    q2, n2, x2, t2 = torch.empty_like(q), torch.empty_like(n), torch.empty_like(x), torch.empty_like(t)
    for turn in range(12):
        for buf in (q2, n2, x2, t2):
            buf.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side if turn % 2 else torch.cuda.current_stream()):
            for _ in range(3):
                slow @ slow
            x2.copy_(x)
            t2.copy_(t)
            n2.copy_(n)
            q2.copy_(q)
            if turn % 3 == 0:
                t2.fill_(3)
                t2[1:].add_(1)
        if turn % 2:
            torch.cuda.current_stream().wait_stream(side)
        r = b.cache.append(n2, n2, q=q2, cos=cos, sin=sin)
        o = b.cache.decode(r) + 0
        p = yr.token_logprobs(x2, t2, top_k=4)
        for got, right in ((r, rotated), (o, want), (p.logprob * 1, lp.logprob), (p.top_token, lp.top_token)):
            assert torch.equal(got, right), turn


FIRST_CALL = """
import torch, yirage_b200 as yr
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
k = torch.randn(5, 64, 2, 128, device="cuda").bfloat16()
cache = yr.PagedKVCache(k, k.clone(), {"qo_indptr_buffer": i32([0, 1]), "paged_kv_indptr_buffer": i32([0, 4]),
                        "paged_kv_indices_buffer": i32([3, 1, 0, 2] * PAGES), "paged_kv_last_page_len_buffer": i32([9])})
q, n, x, t = (torch.randn(1, 8, 128, device="cuda").bfloat16(), torch.randn(1, 2, 128, device="cuda").bfloat16(),
              torch.randn(3, 5000, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    r = cache.append(n, n, q=q)
    o = cache.decode(r)
    p = yr.token_logprobs(x, t, top_k=2)
g.replay()
torch.cuda.synchronize()
r2 = cache.append(n, n, q=q)
assert torch.equal(o, cache.decode(r2)) and torch.equal(p.top_token, yr.token_logprobs(x, t, top_k=2).top_token)
cache.check()
print("fine")
"""


@pytest.mark.parametrize("pages", [1, 1000])      # clusters; equal ranges (the page list could be long)
def test_first_call_of_a_process_may_be_captured(pages):
    import subprocess
    import sys
    out = subprocess.run([sys.executable, "-c", FIRST_CALL.replace("PAGES", str(pages))], capture_output=True, text=True,
                         timeout=200)
    assert out.returncode == 0 and out.stdout.strip() == "fine", out.stderr[-2000:]


def test_empty_calls_and_shared_memory():
    b = Batch([30, 20], [1, 1], seed=50)
    e = torch.empty(0, 2, 128, dtype=BF16, device="cuda")
    assert b.cache.append(e, e, q=torch.empty(0, 8, 128, dtype=BF16, device="cuda")).shape == (0, 8, 128)
    out, lse = b.cache.decode(torch.empty(0, 8, 128, dtype=BF16, device="cuda"), return_lse=True)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    got = yr.token_logprobs(torch.empty(0, 50, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top_k=3)
    assert got.logprob.shape == (0,) and got.top_token.shape == (0, 3)
    q = rnd(gen(51), 2, 8, 128)
    with pytest.raises(N.YpkError, match="out overlaps q"):
        b.cache.decode(q, out=q)
    both = torch.zeros(3, 8, 128, dtype=BF16, device="cuda")
    with pytest.raises(N.YpkError, match="q_out overlaps q"):
        b.cache.append(rnd(gen(52), 2, 2, 128), rnd(gen(52), 2, 2, 128), q=both[:2], q_out=both[1:])
    q.requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        b.cache.decode(q)
    with torch.no_grad():
        b.cache.decode(q)


def prompt_rows(shape, ow, ids):
    """K and V rows of every layer for a prompt as the projections leave them (bf16 pipeline of the
    oracle), and the logits of its positions."""
    n, d = len(ids), shape.head_dim
    cos, sin = O.rope_tables(d, shape.rope_theta, 256)
    x = ow.embed[torch.tensor(ids)].float()
    keys, values = [], []
    for L in ow.layers:
        h = O.rmsnorm(x, L["input_norm"], ow.eps, "bf16")
        q = O.linear(h, L["q"], rounding="bf16").view(n, ow.num_q_heads, d)
        k = O.linear(h, L["k"], rounding="bf16").view(n, ow.num_kv_heads, d)
        v = O.linear(h, L["v"], rounding="bf16").view(n, ow.num_kv_heads, d)
        keys.append(k)
        values.append(v)
        pages = list(range((n + 63) // 64))
        kc = torch.zeros(len(pages), 64, ow.num_kv_heads, d, dtype=BF16)
        a = O.paged_attention_step(q, k, v, kc, torch.zeros_like(kc), pages, n, 64, ow.num_q_heads, ow.num_kv_heads,
                                   cos, sin, "bf16")
        x = O.linear(a.reshape(n, -1), L["o"], residual=x, rounding="bf16")
        h = O.rmsnorm(x, L["post_norm"], ow.eps, "bf16")
        g, u = O.linear(h, L["gate"], rounding="bf16"), O.linear(h, L["up"], rounding="bf16")
        x = O.linear(O.silu_mul(g, u, "bf16"), L["down"], residual=x, rounding="bf16")
    h = O.rmsnorm(x, ow.final_norm, ow.eps, "bf16")
    return keys, values, O.linear(h, ow.lm_head, rounding="bf16")


@pytest.mark.parametrize("max_tokens", [8, 64])
def test_prompts_handed_over_to_the_persistent_kernel(max_tokens):
    """Two requests whose prompts were run elsewhere enter the persistent kernel with their K / V
    rows appended here; every token it samples is the arg-max of a forward pass over the
    request's whole history (or ties with it), and the log probabilities read from its logits
    in place are those of the sampled tokens."""
    shape = llama.LlamaShape(hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=8,
                             num_key_value_heads=2, vocab_size=3000, rms_norm_eps=1e-5)
    w = llama.init_weights(shape, "cuda", 5)
    ow = oracle_weights(shape, w)
    prompts, max_seq = [70, 64], 80
    tokens = torch.zeros(2, max_seq, dtype=torch.int64)
    for r, n in enumerate(prompts):
        tokens[r, :n] = torch.randint(0, 3000, (n,), generator=torch.Generator().manual_seed(r))
    tokens = tokens.cuda()
    ypk, st = llama.build_decode_kernel(shape, w, tokens=tokens, prompt_lengths=i32(prompts), max_num_batched_requests=2,
                                        max_num_batched_tokens=max_tokens, max_num_pages=6, page_size=64)
    steps = [69, 60]           # all but the last token, and all but four
    rows = [prompt_rows(shape, ow, tokens[r, :n].tolist()) for r, n in enumerate(prompts)]
    keys, values = ([torch.cat([rows[r][side][layer][:steps[r]] for r in range(2)]).to(BF16).cuda() for layer in range(2)]
                    for side in (0, 1))
    ypk.reset()
    llama.enter_cached_prompts(ypk, st, steps, keys, values)
    ypk()
    torch.cuda.synchronize()
    status = ypk.status()
    assert status.error == 0 and status.finished == 1
    # the longer way: 70 + the tokens up to max_seq in one iteration each, the other four later
    got = tokens.cpu()
    for r, n in enumerate(prompts):
        _, _, logits = prompt_rows(shape, ow, got[r, :max_seq - 1].tolist())
        for pos in range(n, max_seq):
            row, tok = logits[pos - 1], int(got[r, pos])
            gap = float(row.max() - row[tok])
            assert gap <= O.ATOL + O.RTOL * float(row.abs().max()), f"request {r} position {pos}: {gap:.3f} below the max"
    # the last iteration ran one row: its logits, read in place
    logits = st["tensors"]["argmax_in"]
    lp = ypk.token_logprobs(logits, 1, top_k=5, valid_cols=3000)
    x = ypk.read_tensor(logits)[:1, :3000]
    again = yr.token_logprobs(x, st["meta"]["output_tokens"][:1], top_k=5)
    for a, b in zip(lp, again):
        assert torch.equal(a, b)
    sampled = int(st["meta"]["output_tokens"][0])
    assert lp.top_token[0, 0] == sampled and lp.logprob[0] == lp.top_logprob[0, 0]
    assert abs(float(lp.logprob[0]) - float(torch.log_softmax(x.to(F64), 1)[0, sampled])) <= 2 ** -15 + 2 ** -20
    with pytest.raises(ValueError):
        ypk.token_logprobs(logits, max_tokens + 1)
    ypk.finalize()


@pytest.mark.parametrize("given", [False, True])
def test_log_probabilities_of_the_persistent_kernels_own_logits(given):
    """By default over the vocabulary that the graph samples from: the lm_head of 3000 rows is padded
    to 4096 with rows of zeros, whose logits are no tokens."""
    shape = llama.LlamaShape(hidden_size=512, intermediate_size=1024, num_hidden_layers=1, num_attention_heads=8,
                             num_key_value_heads=2, vocab_size=3000, rms_norm_eps=1e-5)
    tokens = torch.zeros(2, 64, dtype=torch.int64)
    tokens[:, :5] = torch.tensor([[5, 100, 2999, 7, 1], [9, 8, 7, 6, 5]])
    ypk, st = llama.build_decode_kernel(shape, llama.init_weights(shape, "cuda", 5), tokens=tokens.cuda(),
                                        prompt_lengths=i32([5, 5]), max_num_batched_requests=2,
                                        max_num_batched_tokens=8, max_num_pages=2, page_size=64)
    ypk.reset()
    ypk(max_iterations=4)
    torch.cuda.synchronize()
    logits, sampled = st["tensors"]["argmax_in"], st["meta"]["output_tokens"][:2]
    assert logits.dim(1) == 4096
    lp = ypk.token_logprobs(logits, 2, top_k=32, **(dict(tokens=sampled) if given else {}))
    x = ypk.read_tensor(logits)[:2]
    assert (x[:, 3000:] == 0).all()
    want = torch.log_softmax(x[:, :3000].to(F64), 1)
    entropy = -(want.exp() * want).sum(1)
    assert ((lp.entropy.to(F64) - entropy).abs() <= 2 ** -14 * (1 + entropy)).all()
    assert ((lp.logprob.to(F64) - want.gather(1, sampled)[:, 0]).abs() <= 2 ** -15 + 2 ** -19).all()
    assert (lp.top_token < 3000).all() and torch.equal(lp.top_token[:, :1], sampled)
    ypk.finalize()


def check_far_logprobs(x, t, top_k=3):
    """As check_logprobs, for logits far from zero.  With r = fl(m log2 e) the weights are 2^y,
    y = fma(x, log2 e, -r): of the largest logit m it is not 0 but some e, |e| <= E = 1.45 u |m|, which the
    result takes out again.  What is left of it is what numbers of that size are rounded by: log2 s, e
    and their difference, and a factor of y's own rounding in every weight, 8 u E in all; and in
    u / s, sums 2^-16 off each, 2^-15 E.  Beyond 2^30 a weight is 0 or 1 and only log2 of a count is rounded."""
    x64 = x.to(F64)
    want = torch.log_softmax(x64, 1)
    p = want.exp()
    entropy = -torch.where(p > 0, p * want, 0.0).sum(1)
    top = x64.max(1).values.abs()
    counted = top > 2.0 ** 30
    E = torch.where(counted, 0.0, 1.45 * 2 ** -24 * top)
    base = torch.where(counted, 2.0 ** -20, 2.0 ** -15)
    got = yr.token_logprobs(x, t, top_k=top_k)
    at = torch.topk(order_keys(x) * (1 << 20) - torch.arange(x.shape[1], device="cuda"), top_k, 1).indices
    assert torch.equal(got.top_token, at)
    for lp, w in ((got.logprob[:, None], want.gather(1, t[:, None])), (got.top_logprob, want.gather(1, at))):
        lp = lp.to(F64)
        w = torch.where(torch.isinf(w.to(F32)), float("-inf"), w)            # more than fp32 holds
        seen = w > float("-inf")
        assert torch.equal(lp > float("-inf"), seen)
        bound = base[:, None] * (1 + torch.where(counted[:, None] & seen, w.abs().clamp(max=20.0), 0.0)) \
            + (8 * 2 ** -24 * E)[:, None] + 2 ** -22 * w.abs()
        off = (lp - w).abs()
        assert (off <= bound)[seen].all(), f"log probability off by {off[seen].max().item():.3g}"
    off = (got.entropy.to(F64) - entropy).abs()
    bound = torch.where(counted, 2 ** -20 * (1 + entropy), 2 ** -14 * (1 + entropy) + 2 ** -15 * E)
    assert (off <= bound).all(), f"entropy off by {off.max().item():.3g}"


FAR = (100.0, 1000.0, 6e4, 1e6, 5e8, 2.0 ** 30, 1.2e9, 1e10, 1e30)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,vocab", [(3, 9003), (150, 1003), (2, 5)])
def test_logprobs_far_values_in_the_columns_at_the_ends(dtype, rows, vocab):
    """Rows that start off a 16-byte boundary, and a vocabulary that ends inside a vector: single columns at
    both ends.  The largest logit is the first, the last or one in the middle, alone or twice."""
    g = gen(41)
    for first in (0, 1, 3, 7):
        for base in FAR:
            for sign in (1, -1):
                if base > torch.finfo(dtype).max:
                    continue
                store = torch.full((rows, vocab + 8), float("nan"), dtype=dtype, device="cuda")
                x = store[:, first:first + vocab]
                for tops in ((0,), (vocab - 1,), (vocab // 2,), (0, vocab - 1), (0, vocab // 2)):
                    x.copy_(torch.randn(rows, vocab, generator=g, device="cuda") + sign * base)
                    step = (x.float().abs().max() * torch.finfo(dtype).eps).item()
                    x[:, list(tops)] = x.float().max(1, keepdim=True).values.add(max(2.0, 2 * step)).to(dtype)
                    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
                    t[0] = tops[0]
                    check_far_logprobs(x, t)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [1, 150])
def test_logprobs_far_values_to_a_rounding(dtype, rows):
    """Thousands of columns next to the largest logit at every distance from zero, masks below them."""
    g = gen(42)
    big = torch.finfo(dtype).max
    for base in FAR + (2.0 ** 31, 2.3e38, 3.3e38):
        for sign in (1, -1):
            if base > big:
                continue
            x = (torch.randn(rows, 9000, generator=g, device="cuda") + sign * base).clamp(-big, big).to(dtype)
            x[:, 7000:] = -big
            x[:, 8000:] = float("-inf")
            check_far_logprobs(x, torch.randint(0, 9000, (rows,), generator=g, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,heads,dim,page,lengths", [
    (8, 2, 128, 64, [200, 30]), (16, 1, 128, 16, [700]), (8, 2, 256, 64, [333, 20]),               # clusters
    (8, 2, 128, 64, [9000, 40]), (32, 2, 64, 16, [5000, 1, 300]), (16, 2, 256, 3, [4000, 60]),     # ranges
    (4, 4, 128, 16, [(29 * i) % 131 for i in range(165)] + [3000])])                              # by warps
def test_decode_infinities_in_v(dtype, hq, heads, dim, page, lengths):
    """An infinity in V of a seen position is one in its dimension of the output, however small the
    position's weight is; of both signs, or with a NaN, it is a NaN; other dimensions and heads do not
    notice, nor does anybody what lies outside the window or behind the end."""
    g = gen(95)
    b = Batch(lengths, heads=heads, dim=dim, page=page, dtype=dtype, seed=96)
    inf, scale = float("inf"), 0.5          # weights down to e^-100 of the largest
    q = rnd(gen(97), len(lengths), hq, dim, dtype=dtype, scale=3.0)
    picked = [r for r, n in enumerate(lengths) if n >= 20][:6] + [len(lengths) - 1]
    clean = b.v.clone()
    for r in picked:
        n = lengths[r]
        at = b.where(r, torch.randperm(n, generator=g, device="cuda")[:8])
        lo = b.where(r, torch.arange(n, device="cuda"))
        k = b.k[lo].to(F64)
        # the position that weighs least in head 0, and the one that weighs most
        score = torch.einsum("d,ld->l", q[r, 0].to(F64), k[:, 0])
        ends = b.where(r, torch.stack((score.argmin(), score.argmax())))
        for a, (place, (dim0, value)) in enumerate(zip([0, 1, 0, 1, 0, 1], [(0, inf), (0, inf), (9, -inf), (17, inf), (17, -inf),
                                                                        (dim - 1, float("nan"))])):
            b.v[ends[0][place], ends[1][place], 0, dim0] = value
        b.v[at[0][0], at[1][0], heads - 1, 5] = -inf
    out, lse = b.cache.decode(q, return_lse=True, sm_scale=scale)
    b.cache.check()
    group = hq // heads
    for r, n in enumerate(lengths):
        if not n:
            continue
        at = b.where(r, torch.arange(n, device="cuda"))
        v = b.v[at].to(F64)
        want = torch.zeros(heads, dim, dtype=F64, device="cuda")
        up, down, nan = (v == inf).any(0), (v == -inf).any(0), torch.isnan(v).any(0)
        want[up], want[down], want[nan | (up & down)] = inf, -inf, float("nan")
        odd = (up | down | nan).repeat_interleave(group, 0)
        want = want.repeat_interleave(group, 0)
        got = out[r].to(F64)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), r
        assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), r
        if r in picked:
            assert odd.any()
            check_attention(torch.where(odd, 0.0, got).to(dtype), lse[r], q[r], b.k[at],
                            torch.where((up | down | nan)[None], 0.0, clean[at].to(F64)).to(dtype), scale, dtype)
    # the last 5 positions alone, the others holding infinities
    for r in picked:
        at = b.where(r, torch.arange(lengths[r] - 5, device="cuda"))
        b.v[at] = inf
        at = b.where(r, torch.arange(lengths[r] - 5, lengths[r], device="cuda"))
        b.v[at] = clean[at]
    out = b.cache.decode(q, sm_scale=scale, window=5)
    for r in picked:
        at = b.where(r, torch.arange(lengths[r] - 5, lengths[r], device="cuda"))
        check_attention(out[r], None, q[r], b.k[at], b.v[at], scale, dtype)


def test_written_tensors_count_their_versions():
    """What a call writes, autograd takes notice of: a backward pass that saved the old values fails."""
    b = Batch([30, 20], [1, 1], seed=50)
    b.k.nan_to_num_(0.5)
    n, q = rnd(gen(51), 2, 2, 128), rnd(gen(52), 2, 8, 128)
    out = torch.empty_like(q)
    w = torch.ones((), device="cuda", requires_grad=True)
    y = (b.k.float() * w).sum() + (b.k[:1] * w.bfloat16()).float().sum()
    before = [t._version for t in (b.k, b.v, q, out)]
    b.cache.append(n, n, q=q, q_out=q)
    b.cache.decode(q, out=out)
    assert [t._version - o for t, o in zip((b.k, b.v, q, out), before)] == [1, 1, 1, 1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():          # tensors without versions
        c = Batch([30, 20], [1, 1], seed=50)
        p = rnd(gen(52), 2, 8, 128)
        c.cache.decode(c.cache.append(n, n, q=p, q_out=p), out=torch.empty_like(p))
    assert torch.equal(c.cache.decode(p), out)


def test_queries_and_outputs_side_by_side_in_one_buffer():
    """Rows of q and of what is written that alternate in memory without touching."""
    b = Batch([50, 80, 20], [1, 1, 1], heads=2, seed=13)
    g = gen(14)
    cos, sin = tables(128, 128, BF16)
    rows = rnd(g, 3, 2, 4 + 4 + 2, 128)
    q, out, k, v = rows[:, :, :4], rows[:, :, 4:8], rows[:, :, 8], rows[:, :, 9]
    before = rows.clone()
    want = b.cache.append(k, v, q=q.clone(), cos=cos, sin=sin)
    assert b.cache.append(k, v, q=q, q_out=out, cos=cos, sin=sin).data_ptr() == out.data_ptr()
    same = lambda: torch.equal(rows[:, :, :4], before[:, :, :4]) and torch.equal(rows[:, :, 8:], before[:, :, 8:])
    assert torch.equal(out.reshape(3, 8, 128), want) and same()
    want = b.cache.decode(q.clone())
    b.cache.decode(q, out=out)
    assert torch.equal(out, want) and same()
    both = rnd(g, 3, 2, 8, 128)                      # whole heads alternate
    want = b.cache.decode(both[:, 0].clone())
    b.cache.decode(both[:, 0], out=both[:, 1])
    assert torch.equal(both[:, 1], want)
    with pytest.raises(N.YpkError, match="q_out overlaps k or v"):
        b.cache.append(k, v, q=q, q_out=rows[:, :, 5:9], cos=cos, sin=sin)
    same = yr.PagedKVCache(b.k, b.k, b.meta)         # read as K and V alike, not written as both
    assert torch.equal(same.decode(q), yr.PagedKVCache(b.k, b.k.clone(), b.meta).decode(q))
    with pytest.raises(N.YpkError, match="K and V rows"):
        same.append(k, v)


def test_check_misses_nothing_of_another_stream():
    """A bit that a call on another stream sets while check() reads and clears those of this one is in that
    check or in the next one."""
    b = Batch([60, 60], page=16, seed=15)
    q = rnd(gen(16), 2, 8, 128)
    b.meta["paged_kv_last_page_len_buffer"][0] = 17                   # request 0: a table out of order
    b.meta["paged_kv_indices_buffer"][int(b.meta["paged_kv_indptr_buffer"][1])] = -1     # 1: a bad page
    torch.cuda.synchronize()
    side, slow = torch.cuda.Stream(), torch.randn(1024, 1024, device="cuda")
    for turn in range(200):
        with torch.cuda.stream(side):
            for _ in range(turn % 5 + 1):
                slow @ slow
            b.cache.decode(q)
            done = side.record_event()
        found, last = 0, False
        while not last:
            last = done.query()
            b.cache.decode(q[:1])
            with pytest.raises(N.YpkError, match="out of order") as e:
                b.cache.check()
            found += "outside the pool" in str(e.value)
        assert found == 1, turn
    b.cache.check()


@pytest.mark.parametrize("dtype,table,step", [(BF16, F32, 4), (F16, F32, 12), (BF16, BF16, 8), (F16, F16, 24)])
def test_append_table_rows_on_every_16_byte_boundary(dtype, table, step):
    """Tables as a view into wider rows: any row that starts on a 16-byte boundary."""
    b, c = (Batch([30, 7], [10, 7], dtype=dtype, seed=6) for _ in range(2))
    g = gen(7)
    k, v, q = (rnd(g, 17, h, 128, dtype=dtype) for h in (2, 2, 8))
    cos, sin = tables(64, 128, table)
    wide = torch.full((64, 256 + step), float("nan"), dtype=table, device="cuda")
    wide[:, :128], wide[:, 128:256] = cos, sin
    got = c.cache.append(k, v, q=q, cos=wide[:, :128], sin=wide[:, 128:256])
    assert torch.equal(got, b.cache.append(k, v, q=q, cos=cos, sin=sin))
    assert torch.equal(c.k.view(torch.int16), b.k.view(torch.int16))
    odd = torch.zeros(64, 256 + step // 2, dtype=table, device="cuda")
    with pytest.raises(N.YpkError, match="row stride"):
        c.cache.append(k, v, q=q, cos=odd[:, :128], sin=odd[:, 128:256])


def test_append_and_decode_steps_to_a_rounding():
    """The steps of test_append_and_decode_together with the bounds of append and of decode by
    themselves: the attention is that of the query which append returned, over what the cache holds."""
    steps = 20
    cos, sin = tables(256, 128, BF16)
    b, ks, vs, qs = make_steps(20, steps=steps)
    turned = []
    plain = b.cache.append

    def append(*args, **kw):
        turned.append(plain(*args, **kw).clone())
        return turned[-1]

    b.cache.append = append
    start = list(b.lengths)
    outs = decode_loop(b, cos, sin, ks, vs, qs, steps)
    for r in range(3):
        at = b.where(r, torch.arange(b.lengths[r], device="cuda"))
        k, v = b.k[at], b.v[at]
        for i in range(steps):
            n = start[r] + i + 1
            for got, x in ((k[n - 1], ks[i][r]), (turned[i][r], qs[i][r])):
                y, size = rotated64(x[None], None, 0, cos[n - 1:n], sin[n - 1:n])
                bound = half_step(BF16) * (1 + 2 ** -6) * y.abs() + 2 * 3 * 2 ** -24 * size
                assert ((got.to(F64) - y[0]).abs() <= bound[0]).all(), (r, i)
            assert torch.equal(v[n - 1], vs[i][r])
            check_attention(outs[i][r], None, turned[i][r], k[:n], v[:n], 128 ** -0.5, BF16)


@pytest.mark.parametrize("lengths", [[200, 30], [9000, 40], [(29 * i) % 131 for i in range(165)] + [3000]])
def test_decode_infinities_in_k(lengths):
    """A score of -infinity weighs nothing, all of a head's give zeros; one of +infinity gives NaN."""
    b = Batch(lengths, heads=2, page=16, seed=98)
    q = rnd(gen(99), len(lengths), 8, 128)
    q[:, 0::2, 5], q[:, 1::2, 5] = -1.0, 1.0
    r, n = len(lengths) - 1, lengths[-1]
    one = b.where(r, torch.tensor([n // 2], device="cuda"))
    b.k[one[0], one[1], 0, 5] = float("inf")
    out, lse = b.cache.decode(q, return_lse=True)
    assert torch.isnan(out[r, 1:4:2]).all() and torch.isnan(lse[r, 1:4:2]).all()
    rest = torch.cat((torch.arange(n // 2, device="cuda"), torch.arange(n // 2 + 1, n, device="cuda")))
    at = b.where(r, rest)
    check_attention(out[r, 0:4:2], lse[r, 0:4:2], q[r, 0:4:2], b.k[at][:, :1], b.v[at][:, :1], 128 ** -0.5, BF16)
    at = b.where(r, torch.arange(n, device="cuda"))
    check_attention(out[r, 4:], lse[r, 4:], q[r, 4:], b.k[at][:, 1:], b.v[at][:, 1:], 128 ** -0.5, BF16)
    b.k[at[0], at[1], 0, 5] = float("inf")
    out, lse = b.cache.decode(q, return_lse=True)
    assert (out[r, 0:4:2] == 0).all() and (lse[r, 0:4:2] == float("-inf")).all() and torch.isnan(out[r, 1:4:2]).all()
    check_attention(out[r, 4:], lse[r, 4:], q[r, 4:], b.k[at][:, 1:], b.v[at][:, 1:], 128 ** -0.5, BF16)
