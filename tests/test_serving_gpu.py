"""Serving operators on the GPU against plain 64-bit implementations: rope_append, paged_attention, sample_tokens.

Bounds.  u = eps/2 of the type is the relative error of one rounding.  Rotation: one rounding of the result, and float32
errors of the factors (a reduced angle in half turns is rounded once, 2^-25 * pi; sine and cosine to 2 units in the last
place; two products and a sum): together below 8 * 2^-24 * (|x0| + |x1|) * scaling.  Attention: weights are rounded once (their
sum is not), the result once: u * (A + |out|) with A = sum p |v|; scores are float32 sums of D products, off by at most
(D + 4) 2^-24 scale max_j sum_d |q_d k_jd| =: s; a weight's relative error is at most 2 s and that of its exponential and of
the sums, (keys + 16) 2^-23.
The angle position * inv_freq is a 64-bit number: three roundings in the kernel (the product, 1/2pi, turns) and one in the
reference leave it 4 * 2^-53 * position off, which is nothing at 2^20 and 2^-11 at 2^40.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------ rope_append
def within(got, want, bound):
    """Whether |got - want| <= bound everywhere, and how far off it is where not."""
    off = ((got.double() - want).abs() - bound).amax().item() if got.numel() else 0.0
    return off <= 0, off


def rotate64(x, positions, inv_freq, interleaved, scaling):
    x = x.double()
    r = 2 * len(inv_freq)
    a = positions.double()[:, None, None] * inv_freq.double()
    c, s = a.cos() * scaling, a.sin() * scaling
    y, size = x.clone(), torch.zeros_like(x)
    i0 = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    i1 = i0 + (1 if interleaved else r // 2)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    size[..., i0] = size[..., i1] = (x0.abs() + x1.abs()) * scaling
    return y, size


def check_append(n, heads, kv, dim, rotary, interleaved, dtype, page, views=False, layout="head", far=1 << 20, skip=(), scaling=1.25, in_place=False, seed=0):
    from mxfp4 import rope_append, rope_frequencies
    from mxfp4.serving import check_status
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = n // page + 2
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    if views:
        x = rnd(n, (heads + 2 * kv) * dim + 5)
        q, k, v = (x[:, 5 + a * dim:5 + b * dim].view(n, b - a, dim) if n == 1 else x[:, 5 + a * dim:5 + b * dim].unflatten(1, (b - a, dim))
                   for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    else:
        q, k, v = rnd(n, heads, dim), rnd(n, kv, dim), rnd(n, kv, dim)
    if layout == "head":
        kc, vc = rnd(pages, kv, page, dim), rnd(pages, kv, page, dim)
    else:                                                  # tokens of a page outermost, one tensor for both
        both = rnd(pages, 2, page, kv, dim)
        kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    positions = torch.randint(0, far, (n,), generator=g, device="cuda")
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
    for i in skip:
        slots[i] = -1 - i
    inv_freq = rope_frequencies(rotary, device="cuda")[0] if rotary else torch.zeros(0, dtype=torch.float64, device="cuda")
    want_k, want_v = kc.clone(), vc.clone()
    want_q, size_q = rotate64(q, positions, inv_freq, interleaved, scaling)
    turned, size_k = rotate64(k, positions, inv_freq, interleaved, scaling)
    q_in = q.clone()
    out = rope_append(q, k, v, kc, vc, positions, slots, inv_freq, interleaved=interleaved, scaling=scaling, q_out=q if in_place else None)
    check_status()
    u = half_step(dtype)
    if in_place:
        assert out is q
    else:
        assert torch.equal(q, q_in)
    angle = 4 * far * 2.0 ** -53
    ok, off = within(out, want_q, u * want_q.abs() * (1 + 1e-3) + (8 * F32 + angle) * size_q + 1e-30)
    assert ok, off
    keep = slots >= 0
    pg, row = slots[keep] // page, slots[keep] % page
    got = kc[pg, :, row].double()
    ok, off = within(got, turned[keep], u * turned[keep].abs() * (1 + 1e-3) + (8 * F32 + angle) * size_k[keep] + 1e-30)
    assert ok, off
    assert torch.equal(out[..., rotary:], q_in[..., rotary:]) and torch.equal(kc[pg, :, row][..., rotary:], k[keep][..., rotary:])
    want_k[pg, :, row] = kc[pg, :, row]                    # everything else is as it was
    want_v[pg, :, row] = v[keep]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,kv,dim,rotary,page", [(1, 4, 4, 128, 128, 16), (7, 8, 2, 64, 32, 16), (300, 6, 3, 32, 32, 64), (33, 5, 1, 80, 16, 32),
                                                       (5, 2, 2, 128, 0, 16), (9, 3, 1, 40, 10, 48), (2, 1, 1, 6, 6, 1)])
def test_rope_append(n, heads, kv, dim, rotary, page, interleaved, dtype):
    check_append(n, heads, kv, dim, rotary, interleaved, dtype, page, skip=(0,) if n == 7 else ())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append_views_layouts_and_in_place(interleaved):
    check_append(130, 8, 2, 64, 64, interleaved, torch.bfloat16, 16, views=True)
    check_append(130, 8, 2, 64, 64, interleaved, torch.bfloat16, 16, layout="token", in_place=True)
    check_append(41, 8, 2, 128, 64, interleaved, torch.float16, 32, layout="token", views=True)
    check_append(700, 4, 2, 128, 128, interleaved, torch.bfloat16, 128, far=1 << 40, in_place=True)


def test_rope_append_of_nothing_and_of_a_bad_slot():
    from mxfp4 import rope_append
    from mxfp4._capi import MXFP4BackendError
    from mxfp4.serving import check_status
    kc = torch.zeros(2, 1, 16, 32, dtype=torch.bfloat16, device="cuda")
    vc, inv = kc.clone(), torch.ones(16, dtype=torch.float64, device="cuda")
    e = lambda n, h: torch.ones(n, h, 32, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    assert rope_append(e(0, 2), e(0, 1), e(0, 1), kc, vc, i(), i(), inv).shape == (0, 2, 32)
    rope_append(e(2, 2), e(2, 1), e(2, 1), kc, vc, i(0, 0), i(32, 3), inv)             # slot 32 is one past the end
    with pytest.raises(MXFP4BackendError, match="outside the cache"):
        check_status()
    check_status()
    assert vc[0, 0, 3].eq(1).all() and vc.sum() == 32


# ------------------------------------------------------------------------------------------------ paged_attention
def make_cache(pages, kv, page, dim, dtype, g, layout):
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    if layout == "head":
        return rnd(pages, kv, page, dim), rnd(pages, kv, page, dim)
    both = rnd(pages, page, 2, kv, dim)
    return both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)


def attend64(q, kc, vc, table, lens, starts, prefix_pages, prefix, scale):
    """out, lse and the two bounds, sequence by sequence in 64 bits"""
    n, heads, dim = q.shape
    kv = kc.shape[1]
    group = heads // kv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    u = half_step(q.dtype)
    rows = lambda c, pages, m, h: c[pages[:-(-m // c.shape[2])].long(), h].double().reshape(-1, dim)[:m]  # noqa: E731
    for b, length in enumerate(lens):
        m = starts[b + 1] - starts[b]
        for h in range(kv):
            k, v = rows(kc, table[b], length, h), rows(vc, table[b], length, h)
            if prefix:
                k, v = torch.cat([rows(kc, prefix_pages, prefix, h), k]), torch.cat([rows(vc, prefix_pages, prefix, h), v])
            for i in range(m):
                sees = prefix + max(0, length - m + i + 1)
                if sees == 0:
                    continue
                x = q[starts[b] + i, h * group:(h + 1) * group].double()
                s = x @ k[:sees].T * scale
                p = s.softmax(-1)
                at = (starts[b] + i, slice(h * group, (h + 1) * group))
                out[at], lse[at] = p @ v[:sees], s.logsumexp(-1)
                size = p @ v[:sees].abs()
                off = (dim + 4) * F32 * abs(scale) * (x.abs() @ k[:sees].abs().T).amax(-1, keepdim=True)
                tol[at] = u * (1 + 1e-3) * (size + out[at].abs()) + size * (2 * off + 2 * (sees + 16) * F32) + torch.finfo(q.dtype).tiny
                tol_lse[at] = off[:, 0] + 2 * (sees + 16) * F32 + 4 * F32 * lse[at].abs()
    return out, lse, tol, tol_lse


def check_attention(lens, heads, kv, dim, page, dtype, queries=None, prefix=0, layout="head", scale=None, poison=True, seed=0, extra_rows=(0, 0), spare=3):
    from mxfp4 import paged_attention
    from mxfp4.serving import check_status
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pre = -(-prefix // page)
    pages = sum(need) + pre + spare
    kc, vc = make_cache(pages, kv, page, dim, dtype, g, layout)
    places = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1) + 1), 1 << 30, dtype=torch.int32, device="cuda")       # never looked at
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = places[at:at + m]
        at += m
    prefix_pages = places[at:at + pre].contiguous()
    if poison:                                             # behind the last key of a sequence: NaN and infinities
        used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            for j in range(need[b]):
                used[table[b, j].long(), :min(page, n - j * page)] = True
        for j in range(pre):
            used[prefix_pages[j].long(), :min(page, prefix - j * page)] = True
        mask = ~used[:, None, :, None].expand(pages, kv, page, dim)
        kc.masked_fill_(mask, math.nan)
        vc.masked_fill_(mask, math.inf)
    counts = queries if queries is not None else [1] * len(lens)
    starts = [extra_rows[0]]
    for m in counts:
        starts.append(starts[-1] + m)
    rows = starts[-1] + extra_rows[1]
    q = torch.randn(rows, heads, dim, generator=g, device="cuda").to(dtype)
    kw = dict(scale=scale)
    if queries is not None:
        kw["q_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if prefix:
        kw.update(prefix_pages=prefix_pages, prefix_len=torch.tensor([prefix], dtype=torch.int32, device="cuda"))
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = paged_attention(q, kc, vc, table, lens_t, return_lse=True, **kw)
    check_status()
    want, want_lse, tol, tol_lse = attend64(q, kc, vc, table, lens, starts, prefix_pages, prefix, dim ** -0.5 if scale is None else scale)
    ok, off = within(out, want, tol)
    assert ok, off
    assert torch.equal(lse.isinf(), want_lse.isinf())
    fine = ~want_lse.isinf()
    ok, off = within(lse[fine], want_lse[fine], tol_lse[fine])
    assert ok, off
    again = paged_attention(q, kc, vc, table, lens_t, **kw)
    assert torch.equal(again, out)                         # the same bits every time
    if queries is not None:                                # rows of no sequence stay as they are
        given = torch.full_like(q, 7.0)
        assert paged_attention(q, kc, vc, table, lens_t, out=given, **kw) is given
        assert torch.equal(given[starts[0]:starts[-1]], out[starts[0]:starts[-1]])
        assert given[:starts[0]].eq(7).all() and given[starts[-1]:].eq(7).all()
        assert out[:starts[0]].eq(0).all() and out[starts[-1]:].eq(0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (8, 2), (8, 1), (34, 2), (70, 1)])
def test_decode(heads, kv, dim, dtype):
    check_attention([1, 37, 64, 65, 0, 200, 129], heads, kv, dim, 16, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_decode_pages_and_layouts(page, layout):
    check_attention([300, 1, 63, 1025], 8, 4, 64, page, torch.bfloat16, layout=layout)
    check_attention([300, 1, 63, 1025], 4, 4, 128, page, torch.bfloat16, layout=layout, prefix=77)


def test_decode_long_and_lonely():
    check_attention([9001], 4, 1, 128, 64, torch.bfloat16)
    check_attention([5000, 3, 7003], 8, 2, 64, 16, torch.float16, scale=0.3)
    check_attention([0], 4, 2, 64, 16, torch.bfloat16)
    check_attention([0, 0, 0], 4, 2, 64, 16, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("prefix", [1, 64, 500])
@pytest.mark.parametrize("heads,kv", [(4, 4), (16, 2)])
def test_decode_with_a_shared_prefix(heads, kv, prefix, dim, dtype):
    check_attention([1, 40, 0, 128, 17], heads, kv, dim, 16, dtype, prefix=prefix)
    check_attention([70], heads, kv, dim, 32, dtype, prefix=prefix)


def test_decode_of_many_sequences():
    check_attention([(i * 37) % 90 for i in range(170)], 4, 2, 64, 16, torch.bfloat16)
    check_attention([(i * 37) % 90 for i in range(170)], 4, 2, 64, 16, torch.bfloat16, prefix=200)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2)])
@pytest.mark.parametrize("prefix", [0, 130])
def test_ragged_queries(heads, kv, prefix, dim, dtype):
    check_attention([70, 1, 33, 5, 140, 0], heads, kv, dim, 16, dtype, queries=[70, 1, 0, 9, 20, 2], prefix=prefix, extra_rows=(0, 3))


def test_ragged_queries_that_fill_tiles():
    check_attention([300, 5, 260], 2, 1, 128, 64, torch.bfloat16, queries=[300, 5, 131])
    check_attention([300, 5, 260], 2, 1, 128, 64, torch.bfloat16, queries=[300, 5, 131], prefix=333)
    check_attention([200, 300], 4, 1, 64, 16, torch.float16, queries=[200, 257], prefix=10, extra_rows=(2, 5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_full_row_tiles(page, dim, dtype):
    # a prompt whose rows end inside a half tile, one of a single token, one behind earlier keys; group sizes 1, 3 and 16
    check_attention([513, 1, 700], 1, 1, dim, page, dtype, queries=[513, 1, 260])
    check_attention([129, 300], 3, 1, dim, page, dtype, queries=[129, 90], prefix=300)
    check_attention([40, 260, 33], 32, 2, dim, page, dtype, queries=[40, 9, 33], layout="token")
    # more query rows than keys, and none at all: rows that see nothing
    check_attention([5, 0, 64], 4, 1, dim, page, dtype, queries=[150, 130, 64])
    check_attention([5, 0, 64], 4, 1, dim, page, dtype, queries=[150, 130, 64], prefix=129)
    # the batch's rows stacked against the prefix: full tiles, a ragged one, heads that do not divide it
    check_attention([(i * 29) % 70 for i in range(90)], 6, 2, dim, page, dtype, prefix=515)
    check_attention([(i * 29) % 70 for i in range(41)], 22, 2, dim, page, dtype, prefix=128)
    check_attention([7, 9], 70, 1, dim, page, dtype, prefix=1000)


def test_ends_of_the_prefix_and_of_the_sequence_in_the_ring_together():
    # the prefix ends inside a tile and the sequence's own keys one or two tiles on, item after item
    check_attention([33, 1, 403, 130, 250], 32, 8, 64, 16, torch.float16, queries=[33, 1, 403, 130, 250], prefix=1999)
    check_attention([33, 1, 403], 8, 2, 128, 16, torch.bfloat16, queries=[33, 1, 403], prefix=257)


def test_growing_scores_rescale_the_sums():
    """Keys whose scores rise along the sequence raise the running maximum again and again."""
    from mxfp4 import paged_attention
    for heads, rows in ((1, 300), (1, 1)):
        g = torch.Generator(device="cuda").manual_seed(3)
        n, dim, page = 1500, 64, 64
        pages = -(-n // page)
        ramp = torch.linspace(-6, 6, pages * page, device="cuda").view(pages, 1, page, 1)
        kc = (ramp + 0.05 * torch.randn(pages, 1, page, dim, generator=g, device="cuda")).to(torch.bfloat16)
        vc = torch.randn(pages, 1, page, dim, generator=g, device="cuda").to(torch.bfloat16)
        q = (1 + 0.1 * torch.randn(rows, heads, dim, generator=g, device="cuda")).to(torch.bfloat16)
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        kw = dict(q_starts=torch.tensor([0, rows], dtype=torch.int32, device="cuda")) if rows > 1 else {}
        out, lse = paged_attention(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0, return_lse=True, **kw)
        want, want_lse, tol, tol_lse = attend64(q, kc, vc, table, [n], [0, rows], None, 0, 1.0)
        ok, off = within(out, want, tol)
        assert ok, off
        ok, off = within(lse, want_lse, tol_lse)
        assert ok, off


def test_pages_behind_two_to_the_31_elements():
    from mxfp4 import paged_attention, rope_append, rope_frequencies
    from mxfp4.serving import check_status
    pages, kv, page, dim, heads = 2080, 8, 1024, 128, 16
    kc, vc = (torch.empty(pages, kv, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(2)
    table = torch.tensor([[2079, 3], [2060, 2078]], dtype=torch.int32, device="cuda")
    for i in table.flatten().tolist():
        kc[i].normal_(generator=g)
        vc[i].normal_(generator=g)
    rnd = lambda *d: torch.randn(*d, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    q, k, v = rnd(2, heads, dim), rnd(2, kv, dim), rnd(2, kv, dim)
    lens, inv = torch.tensor([1024 + 5, 1024 + 700], dtype=torch.int32, device="cuda"), rope_frequencies(dim, device="cuda")[0]
    slots = torch.tensor([3 * 1024 + 4, 2078 * 1024 + 699], device="cuda")
    positions = lens.long() - 1
    q = rope_append(q, k, v, kc, vc, positions, slots, inv)
    want_k, size = rotate64(k, positions, inv, False, 1.0)
    got_k = torch.stack([kc[3, :, 4], kc[2078, :, 699]])
    ok, off = within(got_k, want_k, half_step(torch.bfloat16) * want_k.abs() * (1 + 1e-3) + 8 * F32 * size)
    assert ok, off
    assert torch.equal(torch.stack([vc[3, :, 4], vc[2078, :, 699]]), v)
    for kw, starts, rows in (({}, [0, 1, 2], q), (dict(q_starts=torch.tensor([0, 70, 140], dtype=torch.int32, device="cuda")), [0, 70, 140], rnd(140, heads, dim))):
        out = paged_attention(rows, kc, vc, table, lens, **kw)
        want, _, tol, _ = attend64(rows, kc, vc, table, lens.tolist(), starts, None, 0, dim ** -0.5)
        ok, off = within(out, want, tol)
        assert ok, off
    check_status()


def test_strided_outputs_and_one_query_for_all():
    from mxfp4 import paged_attention
    g = torch.Generator(device="cuda").manual_seed(4)
    kc, vc = make_cache(12, 2, 32, 64, torch.float16, g, "token")
    table = torch.randperm(12, generator=g, device="cuda").to(torch.int32).view(2, 6)
    lens = torch.tensor([180, 97], dtype=torch.int32, device="cuda")
    one = torch.randn(1, 8, 64, generator=g, device="cuda").to(torch.float16)
    for n, kw, starts in ((2, {}, [0, 1, 2]), (200, dict(q_starts=torch.tensor([0, 103, 200], dtype=torch.int32, device="cuda")), [0, 103, 200])):
        q = one.expand(n, 8, 64)                           # every token the same query, without copies
        wide = torch.full((n, 3, 8, 64), 5.0, dtype=torch.float16, device="cuda")
        paged_attention(q, kc, vc, table, lens, out=wide[:, 1], **kw)
        want, _, tol, _ = attend64(q, kc, vc, table, lens.tolist(), starts, None, 0, 64 ** -0.5)
        ok, off = within(wide[:, 1], want, tol)
        assert ok, off
        assert wide[:, 0].eq(5).all() and wide[:, 2].eq(5).all()


def test_strides_over_a_single_entry_mean_nothing():
    from mxfp4 import paged_attention, rope_append, rope_frequencies
    g = torch.Generator(device="cuda").manual_seed(6)
    odd = lambda t, *st: torch.as_strided(t, t.shape, st)  # noqa: E731
    kc, vc = make_cache(1, 1, 32, 64, torch.bfloat16, g, "head")
    q = torch.randn(1, 1, 64, generator=g, device="cuda").to(torch.bfloat16)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    want = paged_attention(q, kc, vc, table, lens)
    assert torch.equal(paged_attention(odd(q, 3, 5, 1), odd(kc, 1, 7, 64, 1), odd(vc, 0, 9, 64, 1), table, lens), want)
    k, v, inv = torch.randn_like(q), torch.randn_like(q), rope_frequencies(64, device="cuda")[0]
    at = torch.tensor([7], device="cuda")
    turned = rope_append(q, k, v, kc, vc, at, at, inv)
    k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
    assert torch.equal(rope_append(odd(q, 3, 5, 1), odd(k, 1, 1, 1), odd(v, 0, 0, 1), odd(k2, 1, 7, 64, 1), odd(v2, 0, 9, 64, 1), at, at, inv), turned)
    assert torch.equal(k2[0, 0, 7], kc[0, 0, 7]) and torch.equal(v2[0, 0, 7], vc[0, 0, 7])


def test_pages_outside_the_cache_and_bad_lengths_are_reported():
    from mxfp4 import paged_attention
    from mxfp4._capi import MXFP4BackendError
    from mxfp4.serving import check_status
    kc = torch.randn(4, 2, 16, 64, device="cuda").to(torch.bfloat16)
    q = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    good = i(0, 1).view(2, 1)
    for table, lens, kw in [(i(4, 1).view(2, 1), i(3, 3), {}), (i(-1, 1).view(2, 1), i(3, 3), {}), (good, i(17, 3), {}), (good, i(-1, 3), {}),
                            (good, i(3, 3), dict(prefix_pages=i(9), prefix_len=i(5))), (good, i(3, 3), dict(prefix_pages=i(2), prefix_len=i(17))),
                            (good, i(3, 3), dict(q_starts=i(0, 1, 3))), (good, i(3, 3), dict(q_starts=i(1, 0, 2)))]:
        out = paged_attention(q, kc, kc, table, lens, **kw)
        with pytest.raises(MXFP4BackendError):
            check_status()
        assert out.isfinite().all()
    paged_attention(q, kc, kc, good, i(3, 3))
    check_status()


# ------------------------------------------------------------------------------------------------ sample_tokens
def sample64(logits, u, heat, k, p, m):
    """Row by row, as the definition reads."""
    tokens, logprobs = [], []
    for r in range(logits.shape[0]):
        row = torch.nan_to_num(logits[r].double().cpu(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        top = row.max()
        if heat[r] <= 0 or not math.isfinite(top):
            tokens.append(int((row == top).nonzero()[0]))
            logprobs.append(0.0)
            continue
        order = torch.argsort(-row, stable=True)
        x = (row[order] - top) / heat[r]
        w = torch.where(x == -math.inf, 0.0, x.exp())
        if 0 < k[r] < len(w):
            w = w[:k[r]]
        if p[r] < 1:
            w = w[:max(1, int((w.cumsum(0) < p[r] * w.sum()).sum()) + 1)]
        if m[r] > 0:
            w = w[w >= min(m[r], 1.0)]
        c = w.cumsum(0)
        at = min(int((c <= max(u[r], 0.0) * c[-1]).sum()), len(w) - 1)
        # u of 1 and more: the last token that has a weight.  In fixed point, one under 2^-(63 - bits) of the largest has none.
        while float(w[at]) * 2.0 ** (62 - (len(row) - 1).bit_length()) < 0.5:
            at -= 1
        tokens.append(int(order[at]))
        logprobs.append(float(x[at] - c[-1].log()))
    return tokens, logprobs


def check_sample(logits, u, heat=1.0, k=0, p=1.0, m=0.0):
    from mxfp4 import sample_tokens
    rows = logits.shape[0]
    as_list = lambda v: v.tolist() if isinstance(v, torch.Tensor) else [v] * rows  # noqa: E731
    got, lp = sample_tokens(logits, u, temperature=heat, top_k=k, top_p=p, min_p=m, return_logprobs=True)
    tokens, logprobs = sample64(logits, u.double().tolist(), as_list(heat), as_list(k), as_list(p), as_list(m))
    assert got.dtype == torch.int64 and got.tolist() == tokens
    # one float32 rounding of a 64-bit value; fixed-point weights add at most vocab * 2^-38 to the kept sum
    want = torch.tensor(logprobs, dtype=torch.float64)
    ok, off = within(lp.cpu(), want, want.abs() * F32 * 1.01 + logits.shape[1] * 2.0 ** -38)
    assert ok, off


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 17), (9, 1000), (2, 32000), (160, 4097), (1, 131072), (600, 300)])
@pytest.mark.parametrize("setting", [dict(), dict(heat=0.7, k=40, p=0.95), dict(k=1), dict(p=0.5, heat=1.5), dict(m=0.05), dict(k=7, p=0.9, m=0.1), dict(heat=0.0), dict(p=0.0)])
def test_sample(rows, vocab, dtype, setting):
    g = torch.Generator(device="cuda").manual_seed(rows * vocab)
    check_sample((torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype), torch.rand(rows, generator=g, device="cuda"), **setting)


def test_sample_settings_per_row_and_pitch():
    g = torch.Generator(device="cuda").manual_seed(5)
    rows, vocab = 64, 5003
    x = (torch.randn(rows, vocab + 13, generator=g, device="cuda") * 2).to(torch.bfloat16)[:, 3:3 + vocab]
    pick = lambda values, t: torch.tensor(values, dtype=t, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]  # noqa: E731
    check_sample(x, torch.rand(rows, generator=g, device="cuda"), heat=pick([0.0, 0.5, 1.0, 2.0], torch.float32), k=pick([0, 1, 30, 100000], torch.int32),
                 p=pick([0.0, 0.3, 0.9, 1.0], torch.float32), m=pick([0.0, 0.02, 1.0, 3.0], torch.float32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_sample_ties_masks_and_borders(dtype):
    inf = math.inf
    x = torch.zeros(12, 1024)
    x[1, ::2] = -inf                                       # a masked vocabulary
    x[2] = -inf                                            # nothing left
    x[3, 700] = inf
    x[3, 900] = inf
    x[4, :512] = math.nan
    x[5] = math.nan
    x[6, 5:] = -60000.0                                    # far below, in float16 too
    x[7, 1::2] = -0.0                                      # equal to 0
    x[8, 17] = 4.0
    x[9] = torch.linspace(-4, 4, 1024)
    x[10] = -inf
    x[10, 1023] = -3.0
    x[11, 3] = -inf
    x = x.to(dtype).cuda()
    for u in [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0, -1.0]:
        for kw in [dict(), dict(k=10), dict(p=0.5), dict(m=0.5), dict(k=512, p=0.25), dict(heat=0.0), dict(heat=0.01)]:
            check_sample(x, torch.full((12,), u, device="cuda"), **kw)


@pytest.mark.parametrize("dtype,step", [(torch.bfloat16, 2.0 ** -133), (torch.float16, 2.0 ** -24), (torch.float32, 2.0 ** -149)])
def test_sample_subnormal_logits(dtype, step):
    g = torch.Generator(device="cuda").manual_seed(5)
    # whole multiples of the type's least value; a temperature of 16 of them tells their neighbours apart
    logits = (torch.randint(-100, 101, (4, 20000), generator=g, device="cuda").double() * step).to(dtype)
    heat = 16 * step
    u = torch.rand(4, generator=g, device="cuda")
    check_sample(logits, u, torch.full((4,), heat, device="cuda"))
    check_sample(logits, u, torch.full((4,), heat, device="cuda"), p=0.7)
    check_sample(logits, u, torch.full((4,), heat, device="cuda"), k=300)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [1, 9, 10, 32, 33, 74, 75, 222])
def test_sample_rows_shared_by_ctas(rows, dtype):
    # every division of a row among CTAs, rows that do not begin at 16 bytes, dense and thin ends of top-k and top-p, ties over the parts
    g = torch.Generator(device="cuda").manual_seed(rows)
    vocab = 8195
    wide = (torch.randn(rows, vocab + 6, generator=g, device="cuda") * 3).to(dtype)
    wide[rows // 2, 100:] = wide[rows // 2, 100]
    wide[0, 5:5000:7] = float("nan")
    wide[-1, 4000:] = float("-inf")
    logits = wide[:, 3:3 + vocab]
    r = torch.arange(rows)
    check_sample(logits, torch.rand(rows, generator=g, device="cuda"), torch.where(r % 7 == 5, 0.0, 0.5 + r % 3 * 0.7).float().cuda(),
                 (r * 97 % 8000).int().cuda(), (1.0 - r % 5 * 0.2).float().cuda(), (r % 4 * 0.002).float().cuda())
    check_sample(logits, torch.ones(rows, device="cuda"), 1.3, 0, 0.95)


def test_sample_of_nothing():
    from mxfp4 import sample_tokens
    assert sample_tokens(torch.zeros(0, 10, device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)


# ------------------------------------------------------------------------------------------------ streams, captures, together
def step_inputs(seed, batch=5, heads=4, kv=2, dim=64, page=16, vocab=500, prefix=33):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    table = torch.arange(batch * 8, device="cuda", dtype=torch.int32).view(batch, 8) + 3
    return dict(qkv=rnd(batch, (heads + 2 * kv) * dim), kc=rnd(batch * 8 + 3, kv, page, dim), vc=rnd(batch * 8 + 3, kv, page, dim), table=table,
                head=rnd(vocab, heads * dim), lens=torch.randint(1, 100, (batch,), generator=g, device="cuda").to(torch.int32),
                pre=torch.arange(3, device="cuda", dtype=torch.int32), pre_len=torch.tensor([prefix], dtype=torch.int32, device="cuda"),
                u=torch.rand(batch, generator=g, device="cuda"), page=page, heads=heads, kv=kv, dim=dim, batch=batch)


def step(s):
    """One decode step as a model makes it: append, attend, project, sample, and one token on."""
    from mxfp4 import paged_attention, rope_append, rope_frequencies, sample_tokens
    b, h, kv, d = s["batch"], s["heads"], s["kv"], s["dim"]
    x = s["qkv"]
    q, k, v = x[:, :h * d].view(b, h, d), x[:, h * d:(h + kv) * d].view(b, kv, d), x[:, (h + kv) * d:].view(b, kv, d)
    place = s["lens"].long()
    slots = s["table"].long().gather(1, (place // s["page"])[:, None])[:, 0] * s["page"] + place % s["page"]
    if "freq" not in s:
        s["freq"] = rope_frequencies(d, device="cuda")[0]
    q = rope_append(q, k, v, s["kc"], s["vc"], place + s["pre_len"], slots, s["freq"])
    s["lens"].add_(1)
    o = paged_attention(q, s["kc"], s["vc"], s["table"], s["lens"], prefix_pages=s["pre"], prefix_len=s["pre_len"])
    logits = o.reshape(b, h * d) @ s["head"].T
    return o, sample_tokens(logits, s["u"], temperature=0.9, top_k=50, top_p=0.9)


def test_a_step_in_order_against_64_bits():
    s = step_inputs(1)
    first = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    o, token = step(s)
    b, h, kv, d = s["batch"], s["heads"], s["kv"], s["dim"]
    x = first["qkv"]
    pos = first["lens"].long() + first["pre_len"]
    q, _ = rotate64(x[:, :h * d].view(b, h, d), pos, s["freq"], False, 1.0)
    k, _ = rotate64(x[:, h * d:(h + kv) * d].view(b, kv, d), pos, s["freq"], False, 1.0)
    kc, vc = first["kc"].clone(), first["vc"].clone()
    for i in range(b):
        at = int(first["lens"][i])
        kc[first["table"][i, at // 16].long(), :, at % 16] = k[i].to(kc.dtype)
        vc[first["table"][i, at // 16].long(), :, at % 16] = x[i, (h + kv) * d:].view(kv, d)
    q16 = q.to(torch.bfloat16)
    # a rotated element that lies on a border between two bfloat16 values may round the other way: one step of one element
    want, _, tol, _ = attend64(q16, kc, vc, first["table"], (first["lens"] + 1).tolist(), list(range(b + 1)), first["pre"], int(first["pre_len"]), d ** -0.5)
    ok, off = within(o, want, tol + 2.0 ** -7 * tol.amax())
    assert ok, off
    logits = o.reshape(b, h * d) @ s["head"].T
    tokens, _ = sample64(logits, s["u"].double().tolist(), [0.9] * b, [50] * b, [0.9] * b, [0.0] * b)
    assert token.tolist() == tokens


def test_calls_on_two_streams_at_once():
    from mxfp4.serving import check_status
    want = [[tuple(t.clone() for t in step(s)) for _ in range(6)] for s in (step_inputs(21, batch=40), step_inputs(22, batch=3))]
    states, streams, got = [step_inputs(21, batch=40), step_inputs(22, batch=3)], [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(states[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for a, b in zip(got[i], want[i]):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check_status()


def test_captured_steps_follow_their_lengths_and_run_side_by_side():
    from mxfp4.serving import check_status
    eager, graphs, outs, states = [], [], [], []
    for seed in (11, 12):
        s = step_inputs(seed)
        eager.append([tuple(t.clone() for t in step(s)) for _ in range(3)])
        s2 = step_inputs(seed)
        keep = {k: v.clone() for k, v in s2.items() if isinstance(v, torch.Tensor)}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s2)
            for k, v in keep.items():
                s2[k].copy_(v)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step(s2)
        torch.cuda.current_stream().wait_stream(side)
        for k, v in keep.items():
            s2[k].copy_(v)
        graphs.append(g)
        outs.append(out)
        states.append(s2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for j in range(3):
        for i in (0, 1):                                   # two graphs at once, each on a stream of its own
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(outs[i][0], eager[i][j][0]) and torch.equal(outs[i][1], eager[i][j][1]), (i, j)
    check_status()
