"""The paged 8-bit cache: ress_cache_append and ress_cache_attn against 64-bit
references.

Tolerances.  Append: fp32 arithmetic of a few tens of operations on values of
order 1 (1e-5), then one rounding: q to its type (bf16: 2^-9 relative), a code
to e4m3 (half a step: 2^-4 of the value, or 2^-10 of the scale among the
subnormals).  Attention: P is rounded to 16 bits (2^-9 relative at most) in
the numerator and may be in the denominator, so the fp32 output is within
2^-8 sum(p |v|); a quarter of that again covers S and the exponentials in
fp32.  bf16 outputs add 2^-8 of the value."""

import pytest
import torch

from ress_b200 import kernels as K
from ress_b200._lib import RessError

from streaming_ref import (E4M3, E8M0, HD, PAGE, attention, dense_kv, least_scale, make_cache, norm_rotate,
                           shuffled_table)

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tables(n, dtype):
    inv = 1.0 / (100.0 ** (torch.arange(0, 32, 2, device="cuda") / 32))
    ang = torch.outer(torch.arange(n, device="cuda").float(), inv)
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _affine(g):
    return [1 + 0.3 * torch.randn(HD, device="cuda", generator=g), 0.2 * torch.randn(HD, device="cuda", generator=g)]


def _u8(x):
    return x.view(torch.uint8)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _check_stored(cache, table, lens, counts, k, v):
    """The pages hold k, v (fp64, (B, T, H, 64)) behind lens: scales exactly, values to half a step."""
    for name, x in (("k", k), ("v", v)):
        codes, scale = cache[name + "_pages"], _u8(cache[name + "_scale"]).int() - 127
        for b in range(k.shape[0]):
            held, n, at = int(lens[b]), int(counts[b]), 0
            while at < n:
                page, slot = int(table[b, (held + at) // PAGE]), (held + at) % PAGE
                take = min(PAGE - slot, n - at)
                for h in range(k.shape[2]):
                    y = x[b, at:at + take, h]
                    e = int(scale[page, h])
                    if slot == 0:  # nothing older in the page
                        assert e == least_scale(float(y.abs().max())), (name, b, at, h)
                    got = codes[page, h, slot:slot + take].double() * 2.0 ** e
                    tol = torch.maximum(y.abs() * 2.0 ** -4, torch.full_like(y, 2.0 ** (e - 10))) + 1e-5
                    assert bool(((got - y).abs() <= tol).all()), (name, b, at, h)
                at += take


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,Hq,Hkv,held,norm,rope", [
    (1, 1, 2, 2, 0, True, True),        # one token, empty cache
    (1, 1, 2, 2, 63, True, True),       # the last slot of a page
    (1, 1, 3, 1, 64, False, True),      # the first slot of the next
    (3, 5, 6, 2, 62, True, True),       # across a page's end, shared heads
    (2, 64, 4, 4, 0, False, False),     # a whole page, codes only
    (2, 65, 2, 2, 127, True, False),
    (1, 203, 8, 1, 17, True, True),     # four pages and a ragged tail
])
def test_append(dtype, B, T, Hq, Hkv, held, norm, rope):
    g = _gen(B * 1000 + T + held)
    lens = torch.full((B,), held, dtype=torch.int32, device="cuda")
    width = -(-(held + T) // PAGE) + 1
    cache = make_cache(B * width + 3, Hkv)
    table = shuffled_table(B, width, B * width + 3, seed=T)
    # older tokens of small values, so that their page's scale has to grow
    if held:
        old = 0.01 * torch.randn(B, held, Hkv, HD, device="cuda", generator=g)
        K.cache_append(old, 0.5 * old, **cache, table=table, lens=torch.zeros_like(lens))
    before = {n: _u8(t).clone() for n, t in cache.items()}
    qkv = (torch.randn(B, T, Hq + 2 * Hkv, HD, device="cuda", generator=g) * 1.3).to(dtype)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 2)  # views: rows of one projection
    kw = {}
    if norm:
        (kw["qn_weight"], kw["qn_bias"]), (kw["kn_weight"], kw["kn_bias"]) = _affine(g), _affine(g)
    if rope:
        kw["rope_cos"], kw["rope_sin"] = _tables(40, dtype)
        kw["pos"] = torch.randint(-1, 42, (B, T, 2), device="cuda", generator=g)  # out of range: clamped
    out = K.cache_append(k, v, **cache, table=table, lens=lens, q=q, **kw)
    torch.cuda.synchronize()
    assert K.check_status() == 0
    rot = [kw.get("pos"), kw.get("rope_cos"), kw.get("rope_sin")]
    qr = norm_rotate(q, kw.get("qn_weight"), kw.get("qn_bias"), 1e-5, *rot)
    kr = norm_rotate(k, kw.get("kn_weight"), kw.get("kn_bias"), 1e-5, *rot)
    assert out.dtype == dtype and out.shape == q.shape
    tol = 1e-5 + (2.0 ** -8 * qr.abs() if dtype == torch.bfloat16 else 0)
    assert bool(((out.double() - qr).abs() <= tol).all())
    _check_stored(cache, table, lens, [T] * B, kr, v.double())
    # older tokens keep their values to a step of the new scale; slots and pages that got nothing keep their bytes
    for b in range(B):
        for h in range(Hkv):
            now = dense_kv(cache, table, lens, b, h)
            was = dense_kv({n: t.view(E4M3 if "pages" in n else E8M0) for n, t in before.items()}, table, lens, b, h)
            for w, x, y in zip("kv", now, was):
                if held:
                    top = 2.0 ** (float(_u8(cache[w + "_scale"])[table[b].long(), h].max()) - 127)
                    assert bool(((x - y).abs() <= 2.0 ** -10 * top).all())
    used = torch.zeros(B * width + 3, PAGE, dtype=torch.bool, device="cuda")
    for b in range(B):
        for i in range(held + T):
            used[int(table[b, i // PAGE]), i % PAGE] = True
    for w in "kv":
        assert torch.equal(_u8(cache[w + "_pages"]).transpose(1, 2)[~used], before[w + "_pages"].transpose(1, 2)[~used])
        idle = ~used.any(1)
        assert torch.equal(_u8(cache[w + "_scale"])[idle], before[w + "_scale"][idle])


def test_append_in_one_go_or_token_by_token():
    """Without subnormal codes on the way, a page does not depend on how its tokens arrived."""
    g = _gen(3)
    B, T, H = 2, 150, 2
    x = torch.randn(2, B, T, H, HD, device="cuda", generator=g)
    x = torch.where(x >= 0, x + 0.5, x - 0.5) * (1 + torch.arange(T, device="cuda")[:, None, None] / 40)
    table = shuffled_table(B, 4, 9, seed=1)
    a, b = make_cache(9, H), make_cache(9, H)
    K.cache_append(x[0], x[1], **a, table=table, lens=_i32(0, 0))
    for t in range(T):
        K.cache_append(x[0][:, t:t + 1], x[1][:, t:t + 1], **b, table=table, lens=_i32(t, t))
    for n in a:
        assert torch.equal(_u8(a[n]), _u8(b[n])), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,Hq,Hkv", [(40, 70, 16, 16), (64, 130, 12, 6), (3, 3000, 5, 5)])
def test_append_many_pages_equals_stream_by_stream(B, T, Hq, Hkv, dtype):
    """Calls large enough for a CTA to take several heads in turn store the same
    bytes as one call per stream, whose CTAs take fewer."""
    g = _gen(B + T)
    lens = torch.randint(0, 90, (B,), device="cuda", dtype=torch.int32, generator=g)
    width = -(-(90 + T) // PAGE)
    table = shuffled_table(B, width, B * width, seed=T)
    kw = dict(zip(("qn_weight", "qn_bias", "kn_weight", "kn_bias"), _affine(g) + _affine(g)))
    cos, sin = _tables(40, dtype)
    pos = torch.randint(0, 40, (B, T, 2), device="cuda", generator=g)
    q, k, v = torch.randn(B, T, Hq + 2 * Hkv, HD, device="cuda", generator=g).to(dtype).split([Hq, Hkv, Hkv], 2)
    one, each = make_cache(B * width, Hkv), make_cache(B * width, Hkv)
    for n in one:
        each[n].view(torch.uint8).copy_(one[n].view(torch.uint8))
    rows = K.cache_append(k, v, **one, table=table, lens=lens, q=q, pos=pos, rope_cos=cos, rope_sin=sin, **kw)
    for b in range(B):
        s = slice(b, b + 1)
        r = K.cache_append(k[s], v[s], **each, table=table[s], lens=lens[s], q=q[s], pos=pos[s], rope_cos=cos, rope_sin=sin,
                           **kw)
        assert torch.equal(r, rows[s])
    assert K.check_status() == 0
    for n in one:
        assert torch.equal(_u8(one[n]), _u8(each[n])), n


def test_append_ragged_and_idempotent():
    """Streams of unlike length and count (none among them); a repeated call changes nothing."""
    g = _gen(5)
    B, T, H = 4, 70, 2
    lens, n_new = _i32(0, 10, 64, 100), _i32(70, 0, 1, 33)
    table = shuffled_table(B, 4, 16, seed=2)
    cache = make_cache(16, H)
    old = torch.randn(B, 100, H, HD, device="cuda", generator=g)
    K.cache_append(old, old, **cache, table=table, lens=torch.zeros_like(lens), n_new=lens)
    k, v = torch.randn(2, B, T, H, HD, device="cuda", generator=g)
    K.cache_append(k, v, **cache, table=table, lens=lens, n_new=n_new)
    first = {n: _u8(t).clone() for n, t in cache.items()}
    _check_stored(cache, table, lens, n_new, k.double(), v.double())
    K.cache_append(k, v, **cache, table=table, lens=lens, n_new=n_new)
    torch.cuda.synchronize()
    assert K.check_status() == 0
    for n, t in cache.items():
        assert torch.equal(_u8(t), first[n])


def test_append_zeros_and_values_that_are_not_finite():
    cache = make_cache(2, 2)
    table, lens = _i32(1, 0).view(1, 2), _i32(0)
    k = torch.zeros(1, 3, 2, HD, device="cuda")
    v = k.clone()
    v[0, 1, 0, 5] = torch.inf
    k[0, 2, 1, 7] = torch.nan
    K.cache_append(k, v, **cache, table=table, lens=lens)
    ks, vs = _u8(cache["k_scale"])[1].tolist(), _u8(cache["v_scale"])[1].tolist()
    assert ks == [0, 255] and vs == [255, 0]
    assert not _u8(cache["k_pages"])[1, :, :3].any() and not _u8(cache["v_pages"])[1, :, :3].any()
    # the page stays NaN when finite tokens follow
    K.cache_append(torch.ones_like(k), torch.ones_like(v), **cache, table=table, lens=_i32(3))
    assert _u8(cache["k_scale"])[1, 1] == 255 and _u8(cache["v_scale"])[1, 0] == 255
    q = torch.ones(1, 1, 2, HD, device="cuda").bfloat16()
    out = K.cache_attn(q, **cache, table=table, lens=_i32(6))
    assert bool(out.isnan().all())


def test_append_reports_pages_out_of_range():
    cache = make_cache(2, 1)
    before = {n: _u8(t).clone() for n, t in cache.items()}
    k = torch.ones(1, 2, 1, HD, device="cuda")
    for table, lens in ((_i32(2).view(1, 1), _i32(0)), (_i32(-1).view(1, 1), _i32(0)), (_i32(0).view(1, 1), _i32(64)),
                        (_i32(0).view(1, 1), _i32(-5))):
        K.cache_append(k, k, **cache, table=table, lens=lens)
        with pytest.raises(RessError, match="out of range"):
            K.check_status()
    for n, t in cache.items():
        assert torch.equal(_u8(t), before[n])


# ------------------------------------------------------------------ attention
def _filled(B, lens, Hkv, seed, gain=1.4):
    width = -(-max(lens) // PAGE) + 1
    n = B * width + 2
    g = _gen(seed)
    cache = make_cache(n, Hkv)
    table = shuffled_table(B, width, n, seed)
    L = max(max(lens), 1)
    k = torch.randn(B, L, Hkv, HD, device="cuda", generator=g) * gain
    v = torch.randn(B, L, Hkv, HD, device="cuda", generator=g) * torch.exp(
        torch.randn(B, L, 1, 1, device="cuda", generator=g))
    ln = _i32(*lens)
    K.cache_append(k, v, **cache, table=table, lens=torch.zeros_like(ln), n_new=ln)
    return cache, table, ln


def _close(out, ref, size):
    tol = (2.0 ** -8 + 2.0 ** -10) * size
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * ref.abs()
    err = (out.double() - ref).abs()
    assert bool((err <= tol + 1e-30).all()), float((err / (tol + 1e-30)).max())


SHAPES = [
    # B, T, Hq, Hkv, lens
    (1, 1, 1, 1, [1]),
    (1, 1, 2, 2, [63]),
    (1, 1, 2, 1, [64]),
    (1, 1, 4, 2, [65]),
    (3, 1, 6, 2, [1, 700, 129]),
    (2, 8, 2, 2, [640, 17]),
    (1, 5, 6, 1, [1500]),            # 30 rows of one head
    (2, 33, 4, 4, [200, 333]),
    (1, 127, 2, 2, [513]),
    (1, 129, 3, 3, [64]),
    (2, 100, 8, 2, [1031, 100]),     # 400 rows of one head
    (1, 300, 2, 2, [4099]),
    (1, 1, 16, 16, [20000]),
    (1, 1374, 2, 2, [2748]),
]


@pytest.mark.parametrize("B,T,Hq,Hkv,lens", SHAPES)
@pytest.mark.parametrize("out_bf16", [False, True])
def test_attention(B, T, Hq, Hkv, lens, out_bf16):
    cache, table, ln = _filled(B, lens, Hkv, seed=T + Hq + lens[0])
    q = torch.randn(B, T, Hq, HD, device="cuda", generator=_gen(1)).bfloat16()
    ref, size = attention(q, cache, table, ln)
    out = K.cache_attn(q, **cache, table=table, lens=ln, out_bf16=out_bf16)
    again = K.cache_attn(q, **cache, table=table, lens=ln, out_bf16=out_bf16)
    torch.cuda.synchronize()
    assert K.check_status() == 0
    _close(out, ref, size)
    assert torch.equal(out, again)  # no order of arrival in the sums


@pytest.mark.parametrize("B,T,Hq,Hkv,lens", [s for s in SHAPES if s[1] > 1 or s[0] > 1])
@pytest.mark.parametrize("kind", ["causal", "frame", "prefix", "empty", "random"])
def test_attention_limits(B, T, Hq, Hkv, lens, kind):
    cache, table, ln = _filled(B, lens, Hkv, seed=T + Hq)
    g = _gen(2)
    i = torch.arange(T, device="cuda", dtype=torch.int32)
    first = (ln - T)[:, None]
    limits = {"causal": first + i + 1, "frame": first + (i // 7 + 1) * 7, "prefix": (i % 3) * 40 + 0 * first,
              "empty": torch.where(i % 2 == 0, 0, 1 << 30) + 0 * first,
              "random": torch.randint(-5, max(lens) + 99, (B, T), device="cuda", generator=g)}[kind]
    limits = limits.to(torch.int32).contiguous()
    q = torch.randn(B, T, Hq, HD, device="cuda", generator=g).bfloat16()
    ref, size = attention(q, cache, table, ln, limits)
    out = K.cache_attn(q, **cache, table=table, lens=ln, limits=limits, out_bf16=False)
    torch.cuda.synchronize()
    assert K.check_status() == 0
    _close(out, ref, size)
    nothing = torch.minimum(limits, ln[:, None]) <= 0
    assert not out[nothing].any()


def test_attention_empty_streams():
    """A stream that holds nothing, beside one that does: zeros."""
    cache, table, ln = _filled(2, [0, 70], 2, seed=4)
    q = torch.randn(2, 200, 4, HD, device="cuda", generator=_gen(4)).bfloat16()
    for T in (1, 200):
        out = K.cache_attn(q[:, :T], **cache, table=table, lens=ln, out_bf16=False)
        assert not out[0].any() and bool(out[1].any())
        _close(out, *attention(q[:, :T], cache, table, ln))
    assert K.check_status() == 0


@pytest.mark.parametrize("T", [1, 150])
def test_attention_peaked_and_flat_rows(T):
    """Scores over a wide range (one key far above the rest, and none), q of very
    unlike sizes, pages of very unlike value scales."""
    B, H, L = 1, 2, 900
    g = _gen(6)
    cache = make_cache(20, H)
    table, ln = shuffled_table(B, 15, 20, seed=6), _i32(L)
    k = torch.randn(B, L, H, HD, device="cuda", generator=g)
    v = torch.randn(B, L, H, HD, device="cuda", generator=g)
    v = v * torch.exp2(torch.randint(-30, 20, (B, L // 60 + 1, H, 1), device="cuda", generator=g).float()
                       ).repeat_interleave(60, 1)[:, :L]
    K.cache_append(k, v, **cache, table=table, lens=_i32(0))
    q = torch.randn(B, T, H, HD, device="cuda", generator=g) * torch.exp2(
        torch.arange(T, device="cuda").float() % 9 - 5)[:, None, None]
    q[:, T // 2] = 0
    q[:, T // 3, :, 1:] *= 1e-4  # one large element among small ones
    q = q.bfloat16()
    out = K.cache_attn(q, **cache, table=table, lens=ln, out_bf16=False)
    _close(out, *attention(q, cache, table, ln))
    assert K.check_status() == 0


@pytest.mark.parametrize("T", [1, 140])
def test_attention_nan_stays_where_it_is_seen(T):
    """Queries that do not see a NaN page are untouched by it; those that do give NaN."""
    cache, table, ln = _filled(1, [300], 2, seed=8)
    _u8(cache["v_scale"])[table[0, 3].long(), 0] = 255
    _u8(cache["k_scale"])[table[0, 2].long(), 1] = 255
    q = torch.randn(1, T, 2, HD, device="cuda", generator=_gen(8)).bfloat16()
    for limit, bad in ((128, (False, False)), (129, (False, True)), (193, (True, True))):
        limits = torch.full((1, T), limit, dtype=torch.int32, device="cuda")
        if T > 1:
            limits[0, 0] = 300  # one query of the same tile sees everything
        out = K.cache_attn(q, **cache, table=table, lens=ln, limits=limits, out_bf16=False)
        rest = out[:, 1:] if T > 1 else out
        for h in range(2):
            assert bool(rest[:, :, h].isnan().all()) == bad[h] and bool(rest[:, :, h].isnan().any()) == bad[h]
        if T > 1:
            assert bool(out[:, 0].isnan().all())
    K.check_status()


def test_attention_strides_scale_and_output():
    """q rows out of a wider tensor, pages out of a pool that holds k and v together, out into a wider tensor."""
    B, T, H, L = 2, 37, 3, 500
    g = _gen(9)
    pool = torch.zeros(20, 2, H, PAGE, HD, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(20, 2, H, dtype=torch.uint8, device="cuda")
    cache = dict(k_pages=pool[:, 0].view(E4M3), v_pages=pool[:, 1].view(E4M3), k_scale=scales[:, 0].view(E8M0),
                 v_scale=scales[:, 1].view(E8M0))
    table, ln = shuffled_table(B, 9, 20, seed=9), _i32(L, L - 77)
    k, v = torch.randn(2, B, L, H, HD, device="cuda", generator=g)
    K.cache_append(k, v, **cache, table=table, lens=_i32(0, 0), n_new=ln)
    wide = torch.randn(B, H, T, 2 * HD, device="cuda", generator=g).bfloat16()
    q = wide[..., HD:].transpose(1, 2)  # (B, T, H, 64), heads outside tokens
    out = torch.full((B, T, H + 1, HD), 7.0, device="cuda")
    got = K.cache_attn(q, **cache, table=table, lens=ln, sm_scale=0.3, out=out[:, :, :H])
    assert got.data_ptr() == out.data_ptr()
    _close(out[:, :, :H], *attention(q, cache, table, ln, sm_scale=0.3))
    assert bool((out[:, :, H] == 7).all())
    plain = K.cache_attn(q.contiguous(), **cache, table=table, lens=ln, sm_scale=0.3, out_bf16=False)
    assert torch.equal(plain, out[:, :, :H])


def test_attention_reports_lengths_and_pages_out_of_range():
    cache, table, ln = _filled(1, [100], 1, seed=10)
    q = torch.randn(1, 1, 1, HD, device="cuda", generator=_gen(1)).bfloat16()
    width = table.shape[1]
    for lens, tab in ((_i32(64 * width + 1), table), (_i32(-1), table), (ln, torch.full_like(table, 1000)),
                      (ln, torch.full_like(table, -1))):
        out = K.cache_attn(q, **cache, table=tab, lens=lens)
        with pytest.raises(RessError, match="out of range"):
            K.check_status()
        if lens is ln:
            assert bool(out.isnan().all())
    many = q.expand(1, 130, 1, HD)
    out = K.cache_attn(many, **cache, table=torch.full_like(table, 1000), lens=ln)
    assert bool(out.isnan().all())
    with pytest.raises(RessError, match="out of range"):
        K.check_status()


def test_other_stream_and_graph():
    """The calls run on the current stream and can be captured in a graph."""
    B, H, L = 1, 4, 200
    g = _gen(11)
    cache, table = make_cache(8, H), shuffled_table(B, 6, 8, seed=11)
    k, v = torch.randn(2, B, L, H, HD, device="cuda", generator=g)
    q = torch.randn(B, 5, H, HD, device="cuda", generator=g).bfloat16()
    lens, held = _i32(0), _i32(L)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.cache_append(k, v, **cache, table=table, lens=lens)
        out = K.cache_attn(q, **cache, table=table, lens=held)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.cache_append(k, v, **cache, table=table, lens=lens)
        captured = K.cache_attn(q, **cache, table=table, lens=held)
    for t in cache.values():
        _u8(t).fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, out)
    assert K.check_status() == 0


def test_refusals():
    cache, table, ln = _filled(1, [10], 2, seed=12)
    k = torch.zeros(1, 3, 2, HD, device="cuda")
    q = torch.zeros(1, 3, 4, HD, device="cuda", dtype=torch.bfloat16)
    ok = dict(**cache, table=table, lens=ln)

    def refuse(f, *args, **kw):
        with pytest.raises(RessError):
            f(*args, **{**ok, **kw})

    refuse(K.cache_attn, q.float())
    refuse(K.cache_attn, q.cpu())
    refuse(K.cache_attn, q[..., :32])
    refuse(K.cache_attn, q[:, :, :3])                                    # 3 heads over 2
    refuse(K.cache_attn, q, table=table.long())
    refuse(K.cache_attn, q, lens=ln.long())
    refuse(K.cache_attn, q, lens=ln.cpu())
    refuse(K.cache_attn, q, limits=torch.zeros(1, 3, device="cuda"))
    refuse(K.cache_attn, q, limits=torch.zeros(1, 4, dtype=torch.int32, device="cuda"))
    refuse(K.cache_attn, q, k_pages=_u8(cache["k_pages"]))
    refuse(K.cache_attn, q, k_scale=_u8(cache["k_scale"]))
    refuse(K.cache_attn, q, v_pages=cache["v_pages"][:, :1])
    refuse(K.cache_attn, q, v_pages=cache["v_pages"].transpose(2, 3))
    refuse(K.cache_attn, q, out=torch.zeros_like(q, dtype=torch.float16))
    odd = torch.zeros(1, 3, 4, HD + 4, device="cuda", dtype=torch.bfloat16)[..., 4:]  # rows 8 bytes off
    refuse(K.cache_attn, odd)
    refuse(K.cache_append, k.half(), k.half())
    refuse(K.cache_append, k, k.bfloat16())
    refuse(K.cache_append, k[:, :, :1], k[:, :, :1])
    refuse(K.cache_append, k, k, q=q)                                    # bf16 q beside fp32 k
    refuse(K.cache_append, k, k, n_new=_i32(1, 2))
    refuse(K.cache_append, k, k, kn_weight=torch.ones(HD, device="cuda"))
    refuse(K.cache_append, k, k, rope_cos=torch.ones(4, 32, device="cuda"))
    cs = torch.ones(4, 32, device="cuda")
    refuse(K.cache_append, k, k, rope_cos=cs, rope_sin=cs)               # no positions
    refuse(K.cache_append, k, k, rope_cos=cs, rope_sin=cs, pos=torch.zeros(1, 3, 2, device="cuda"))
    K.cache_append(k[:, :0], k[:, :0], **ok)                             # nothing to do
    assert K.cache_attn(q[:, :0], **ok).shape == (1, 0, 4, HD)
    assert K.check_status() == 0


@pytest.mark.parametrize("T", [1, 3, 12, 40])
@pytest.mark.parametrize("gap,weight", [(12, -80), (40, -80), (40, -40), (100, -100), (100, -150)])
def test_attention_value_scales_far_apart(T, gap, weight):
    """Pages whose values are 2^gap times the others' and whose weights are
    2^weight of theirs: what a page adds does not depend on the scales of pages
    seen before it.  The heads are enough for a warp of the few-query kernel to
    take pages 8 apart in turn: small values, large ones, small ones again."""
    H, pages = 300, 24
    g = _gen(T + gap)
    cache, table, ln = make_cache(pages, H), shuffled_table(1, pages, pages, seed=gap), _i32(64 * pages)
    big = table[0, 8:16].long()
    k = torch.zeros(pages, H, PAGE, HD, device="cuda")
    k[big, :, :, 0] = -240.0
    k[..., 1:] = 0.05 * torch.randn(pages, H, PAGE, HD - 1, device="cuda", generator=g)
    cache["k_pages"].copy_(k)
    cache["v_pages"].copy_(8 * torch.randn(pages, H, PAGE, HD, device="cuda", generator=g))
    for n in ("k_scale", "v_scale"):
        _u8(cache[n]).fill_(127)
    _u8(cache["v_scale"])[big] = 127 + gap
    q = torch.randn(1, T, H, HD, device="cuda", generator=g)
    q[..., 0] = -weight * 0.6931 * 8 / 240
    q = q.bfloat16()
    out = K.cache_attn(q, **cache, table=table, lens=ln, out_bf16=False)
    torch.cuda.synchronize()
    assert K.check_status() == 0
    _close(out, *attention(q, cache, table, ln))


@pytest.mark.parametrize("T", [1, 12, 140])
@pytest.mark.parametrize("code", [0x7F, 0xFF])
def test_attention_nan_codes(T, code):
    """A NaN among a value's codes shows in its dim of the rows that see it, and
    nowhere else; one in a key makes those rows NaN."""
    L, H = 300, 2
    cache, table, ln = _filled(1, [L], H, seed=13)
    q = torch.randn(1, T, H, HD, device="cuda", generator=_gen(13)).bfloat16()
    limits = torch.full((1, T), L, dtype=torch.int32, device="cuda")
    if T > 1:
        limits[0, 1::4], limits[0, 2::4], limits[0, 3::4] = 100, 128, 111
    ref, size = attention(q, cache, table, ln, limits)
    want = torch.zeros_like(ref, dtype=torch.bool)
    for token, head, dim, key in ((30, 0, 5, False), (110, 1, 63, False), (110, 1, 8, False), (150, 0, 17, False),
                                  (299, 1, 40, False), (299, 0, 3, True)):
        pages = _u8(cache["k_pages" if key else "v_pages"])
        pages[table[0, token // PAGE].long(), head, token % PAGE, dim] = code
        sees = limits[0] > token
        want[0, sees, head] |= True if key else (torch.arange(HD, device="cuda") == dim)
        out = K.cache_attn(q, **cache, table=table, lens=ln, limits=limits if T > 1 else None, out_bf16=False)
        torch.cuda.synchronize()
        assert torch.equal(out.isnan(), want), (token, head, dim)
        zero = torch.zeros_like(ref)
        _close(out.masked_fill(want, 0), torch.where(want, zero, ref), size)
    assert K.check_status() == 0


def test_attention_takes_queries_of_any_size():
    """bf16 rows up to the largest finite value."""
    cache, table, ln = _filled(1, [200], 2, seed=15, gain=1e-30)
    for T in (1, 9, 150):
        q = torch.randn(1, T, 2, HD, device="cuda", generator=_gen(15))
        q = (q / q.abs().amax(-1, keepdim=True) * 3.3e38).bfloat16()
        out = K.cache_attn(q, **cache, table=table, lens=ln, sm_scale=1e-8, out_bf16=False)
        _close(out, *attention(q, cache, table, ln, sm_scale=1e-8))
    assert K.check_status() == 0


def test_append_refuses_a_pool_without_heads():
    cache, table, ln = _filled(1, [10], 2, seed=14)
    none = {n: t[:, :0] for n, t in cache.items()}
    k = torch.zeros(1, 3, 0, HD, device="cuda")
    with pytest.raises(RessError):
        K.cache_append(k, k, **none, table=table, lens=ln, q=torch.zeros(1, 3, 4, HD, device="cuda"))


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_long_runs_of_a_warp(T, masked):
    """Few queries of so many streams and heads that pages are not split: 75 pages
    a warp, whose ids and scales are fetched 32 at a time."""
    B, H, pages = 20, 16, 600
    cache, table, _ = _filled(1, [64 * pages], H, seed=16)
    g = _gen(16)
    # the streams read one pool, each in its own order
    table = torch.stack([table[0, torch.randperm(pages, generator=g, device="cuda")] for _ in range(B)]).contiguous()
    lens = torch.randint(60 * pages, 64 * pages + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    limits = None
    if masked:
        limits = torch.randint(0, 64 * pages, (B, T), device="cuda", generator=g, dtype=torch.int32)
    q = torch.randn(B, T, H, HD, device="cuda", generator=g).bfloat16()
    out = K.cache_attn(q, **cache, table=table, lens=lens, limits=limits, out_bf16=False)
    torch.cuda.synchronize()
    assert K.check_status() == 0
    _close(out, *attention(q, cache, table, lens, limits))


@pytest.mark.parametrize("kind", ["whole", "random", "steps"])
def test_attention_long_runs_of_a_cta(kind):
    """Many queries of one head: 86 pages a CTA, through every ring several times, without
    masks, with masks on every page, and with both in turn."""
    T, pages = 40 * 256, 600
    cache, table, ln = _filled(1, [64 * pages - 5], 1, seed=17)
    g = _gen(17)
    i = torch.arange(T, device="cuda", dtype=torch.int32)
    limits = {"whole": None, "random": torch.randint(0, 64 * pages, (1, T), device="cuda", generator=g, dtype=torch.int32),
              "steps": (i // 256 * 960 + 100)[None].contiguous()}[kind]
    q = torch.randn(1, T, 1, HD, device="cuda", generator=g).bfloat16()
    out = K.cache_attn(q, **cache, table=table, lens=ln, limits=limits, out_bf16=False)
    torch.cuda.synchronize()
    assert K.check_status() == 0
    _close(out, *attention(q, cache, table, ln, limits))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_norms_of_either_type(dtype):
    """bf16 norms, norms of both types and norms off a 16-byte boundary give the bits of the same values in fp32."""
    g = _gen(18)
    names = ("qn_weight", "qn_bias", "kn_weight", "kn_bias")
    norms = [w.bfloat16() for w in _affine(g) + _affine(g)]
    q, k, v = torch.randn(2, 70, 6, HD, device="cuda", generator=g).to(dtype).split([2, 2, 2], 2)
    table, lens = shuffled_table(2, 2, 5, seed=18), _i32(0, 30)

    def off(w):
        return torch.cat([w[:1], w])[1:]

    results = []
    for kinds in ([w.float() for w in norms], norms, [norms[0], norms[1].float(), norms[2], norms[3].float()],
                  [off(w) for w in norms], [off(w.float()) for w in norms]):
        cache = make_cache(5, 2)
        rows = K.cache_append(k, v, **cache, table=table, lens=lens, q=q, **dict(zip(names, kinds)))
        results.append([rows] + [_u8(t) for t in cache.values()])
    assert K.check_status() == 0
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
