"""The 8-bit streaming operators, measured: frames reach a model one after
another, their keys and values stay in a paged 8-bit cache.

Three operators make one layer of such a run:
  append     q/k LayerNorm and the 2-D rotary embedding of the new tokens,
             their keys and values written into the pages of a cache
             (e4m3, one power-of-two scale per page of 64 tokens and head);
  attention  queries against that cache;
  linear     a Linear layer in 8-bit integers, one scale per token and one
             per output channel.

``run`` computes them by plain torch operations in fp32, or with ``own`` by
the calls a user makes.  Sizes are those of the 518 x 518 aggregator (16
heads of 64, 1374 tokens a frame: 5 special, 37 x 37 patches; widths 1024
and 4096; 1 to 32 views) and of its 24-head relative, with odd ones beside.
"""

import math

import torch

own = False

PAGE = 64  # tokens per page
HD = 64    # head dimension
FRAME = 1374
E4M3_TOP = 0.875 * 2.0 ** 9  # 448, the largest e4m3 value


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token through the first MLP layer: the latency of a call
        dict(name="linear one token", op="linear", m=1, k=1024, n=4096, act="", dtype="bf16"),
        # the special tokens of 33 views, fp32 activations, a head of odd width
        dict(name="linear special tokens", op="linear", m=165, k=1536, n=1000, act="", dtype="fp32"),
        # one frame through the first MLP layer, GELU in the same call
        dict(name="linear frame", op="linear", m=FRAME, k=1024, n=4096, act="gelu", dtype="bf16"),
        # 32 views through the second MLP layer
        dict(name="linear views", op="linear", m=32 * FRAME, k=4096, n=1024, act="", dtype="bf16"),
        # one token added to one stream, inside a page
        dict(name="append one token", op="append", b=1, t=1, hq=16, hkv=16, held=FRAME, norm=True, ragged=False,
             dtype="bf16"),
        # the special tokens of a frame added to 24 streams of unlike length, heads shared by three, no norms
        dict(name="append streams", op="append", b=24, t=5, hq=24, hkv=8, held=300, norm=False, ragged=True,
             dtype="fp32"),
        # one frame added after two
        dict(name="append frame", op="append", b=1, t=FRAME, hq=16, hkv=16, held=2 * FRAME, norm=True, ragged=False,
             dtype="bf16"),
        # 32 views into an empty cache
        dict(name="append views", op="append", b=1, t=32 * FRAME, hq=16, hkv=16, held=0, norm=True, ragged=False,
             dtype="bf16"),
        # one query over eight frames
        dict(name="attend one token", op="attend", b=1, t=1, hq=16, hkv=16, held=8 * FRAME, mask="", ragged=False),
        # one query for each of 16 streams of unlike length, heads shared by three
        dict(name="attend streams", op="attend", b=16, t=1, hq=24, hkv=8, held=32 * FRAME, mask="", ragged=True),
        # the newest of eight frames over all of them
        dict(name="attend frame", op="attend", b=1, t=FRAME, hq=16, hkv=16, held=8 * FRAME, mask="", ragged=False),
        # the newest four of 32 frames, each of them seeing the frames up to its own
        dict(name="attend views", op="attend", b=1, t=4 * FRAME, hq=16, hkv=16, held=32 * FRAME, mask="frame",
             ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "append", "attend"])
    hq, hkv = rng.choice([(16, 16), (24, 24), (24, 8), (16, 4), (8, 1), (3, 3)])
    if op == "linear":
        k, n = 16 * _log(rng, 16, 256), 8 * _log(rng, 16, 512)
        top = min(32 * FRAME, 32 * FRAME * 4096 * 1024 // (k * n))
        return dict(op=op, m=_log(rng, 1, top), k=k, n=n, act=rng.choice(["", "gelu"]),
                    dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if op == "append":
        b = _log(rng, 1, 32)
        # tokens x heads and what the pool holds stay below those of 32 views
        t = _log(rng, 1, max(1, 32 * FRAME * 16 // (b * hq) // 2))
        held = rng.choice([0, _log(rng, 1, max(1, 8192 // b))])
        return dict(op=op, b=b, t=t, hq=hq, hkv=hkv, held=held, norm=rng.random() < 0.5, ragged=b > 1,
                    dtype=rng.choice(["bf16", "bf16", "fp32"]))
    b = _log(rng, 1, 16)
    held = _log(rng, 1, 32 * FRAME)
    room = 16 * 4 * FRAME * 32 * FRAME // (b * hq * held)
    t = rng.choice([1, _log(rng, 1, max(1, min(held, 4 * FRAME, room)))])
    mask = rng.choice(["", "causal", "frame"]) if t > 1 else ""
    return dict(op=op, b=b, t=t, hq=hq, hkv=hkv, held=held, mask=mask, ragged=b > 1)


# ------------------------------------------------------------------ inputs
def _dtype(case):
    return {"bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]


def _pages(tokens):
    return -(-tokens // PAGE)


def _scale_codes(amax):
    """The e8m0 code u (scale 2^(u - 127)) of the smallest power of two that
    brings amax to at most 448; 255 (NaN) where amax is not finite."""
    m, x = torch.frexp(amax)
    u = (x - 9 + (m > 0.875).to(x.dtype) + 127).clamp(0, 254)
    u = torch.where(amax > 0, u, torch.zeros_like(u))
    return torch.where(torch.isfinite(amax), u, torch.full_like(u, 255)).to(torch.int32)


def _scale_values(u):
    """2^(u - 127) as fp32; NaN for 255."""
    bits = torch.where(u == 0, torch.full_like(u, 0x00400000), u << 23)
    return torch.where(u == 255, torch.full_like(u, 0x7FC00000), bits).view(torch.float32)


def _scale_inverse(u):
    """2^(127 - u) as fp32; 0 for 255, so that a page of NaN scale holds zeros."""
    return torch.where(u == 255, torch.zeros_like(u), (254 - u) << 23).view(torch.float32)


def _rotary_tables(n, dtype):
    inv = 1.0 / (100.0 ** (torch.arange(0, 32, 2, device="cuda", dtype=torch.float32) / 32))
    ang = torch.outer(torch.arange(n, device="cuda", dtype=torch.float32), inv)
    ang = torch.cat([ang, ang], dim=-1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _lens(case, g):
    """Tokens that each stream holds: `held`, or between a quarter of it and all of it."""
    b, held = case["b"], case["held"]
    if not case["ragged"] or held == 0:
        return torch.full((b,), held, dtype=torch.int32, device="cuda")
    lo = max(1, held // 4)
    lens = torch.randint(lo, held + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    lens[-1] = held
    return lens


def _pool(b, width, hkv, g):
    """A cache whose pages lie in no order: pages, scales and the table of each stream's pages."""
    n = b * width
    table = torch.randperm(n, generator=g, device="cuda").to(torch.int32).view(b, width)
    cache = {"table": table}
    for name, gain in (("k", 1.4), ("v", 1.0)):
        codes = torch.empty(n, hkv, PAGE, HD, dtype=torch.float8_e4m3fn, device="cuda")
        scale = torch.empty(n, hkv, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (hkv * PAGE * HD))
        for at in range(0, n, step):
            x = gain * torch.randn(min(step, n - at), hkv, PAGE, HD, generator=g, device="cuda")
            x *= torch.randn(x.shape[0], hkv, 1, 1, generator=g, device="cuda").mul_(0.3).exp_()
            u = _scale_codes(x.abs().amax((-1, -2)))
            codes[at:at + step] = (x * _scale_inverse(u)[..., None, None]).to(torch.float8_e4m3fn)
            scale[at:at + step] = u.to(torch.uint8)
        cache[name + "_pages"], cache[name + "_scale"] = codes, scale.view(torch.float8_e8m0fnu)
    return cache


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        # activations as behind a LayerNorm: a few channels far above the rest
        x = normal(m, k) * (0.5 + normal(k).abs()) + 0.3 * normal(k)
        w = normal(n, k) * (0.02 * (0.5 + normal(n, 1).abs()))
        scale = w.abs().amax(-1) / 127.0
        w8 = torch.round(w / scale[:, None]).to(torch.int8)
        return dict(op="linear", act=case["act"], x=x.to(_dtype(case)), w8=w8, w_scale=scale, bias=0.1 * normal(n))

    b, t, hq, hkv = case["b"], case["t"], case["hq"], case["hkv"]
    lens = _lens(case, g)
    if case["op"] == "append":
        dtype = _dtype(case)
        # room for what is held, for t more, and for a page of spare
        cache = _pool(b, _pages(case["held"] + t) + 1, hkv, g)
        state = dict(op="append", lens=lens, n_new=None, norm=None, **cache)
        # one Linear's output, token-major: heads of q, then of k, then of v
        qkv = (normal(b, t, hq + 2 * hkv, HD) * 1.2 + 0.1 * normal(hq + 2 * hkv, HD)).to(dtype)
        state["q"], state["k"], state["v"] = qkv.split([hq, hkv, hkv], dim=2)
        if case["ragged"]:
            state["n_new"] = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        if case["norm"]:
            state["norm"] = tuple(f(normal(HD)) for f in (lambda x: 1 + 0.3 * x, lambda x: 0.2 * x) * 2)
        state["pos"] = torch.randint(0, 38, (b, t, 2), generator=g, device="cuda")
        state["cos"], state["sin"] = _rotary_tables(64, dtype)
        return state

    # one spare page a stream: a table is as long as the longest stream may get
    cache = _pool(b, _pages(case["held"]) + 1, hkv, g)
    limits = None
    if case["mask"]:
        # query i is the stream's token len - t + i: it sees what came up to itself, or up to its frame's end
        i = torch.arange(t, device="cuda", dtype=torch.int32)
        group = 1 if case["mask"] == "causal" else FRAME
        first = lens[:, None] - t
        limits = torch.minimum(first + (i // group + 1) * group, lens[:, None]).clamp_(min=0).contiguous()
    q = (normal(b, t, hq, HD) * (0.5 + normal(hq, 1).abs())).bfloat16()
    return dict(op="attend", q=q, lens=lens, limits=limits, **cache)


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return {"linear": _own_linear, "append": _own_append, "attend": _own_attend}[s["op"]](s)
    return {"linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[s["op"]](s)


def _own_linear(s):
    from ress_b200 import kernels as K

    return K.int8_linear(s["x"], s["w8"], s["w_scale"], s["bias"], act=s["act"] or None)


def _own_append(s):
    from ress_b200 import kernels as K

    norm = s["norm"] or (None,) * 4
    q = K.cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                       q=s["q"], n_new=s["n_new"], qn_weight=norm[0], qn_bias=norm[1], kn_weight=norm[2],
                       kn_bias=norm[3], pos=s["pos"], rope_cos=s["cos"], rope_sin=s["sin"])
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _own_attend(s):
    from ress_b200 import kernels as K

    return K.cache_attn(s["q"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                        limits=s["limits"])


def _plain_linear(s):
    x = s["x"].float()
    scale = x.abs().amax(-1, keepdim=True) * (1.0 / 127.0)
    x8 = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale)))
    y = (x8 @ s["w8"].float().t()) * scale * s["w_scale"] + s["bias"]
    if s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y.to(s["x"].dtype)


def _plain_prologue(x, weight, bias, s):
    """LayerNorm over the head dimension (where there is one), then the rotary embedding, in fp32."""
    x = x.float()
    if weight is not None:
        x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * weight + bias
    # (B, T, 1, 64): dims 0-31 turn by the row, 32-63 by the column
    cos, sin = (tab.float()[s["pos"]].flatten(-2)[:, :, None] for tab in (s["cos"], s["sin"]))
    a, b = x.unflatten(-1, (2, 2, 16)).unbind(-2)
    turned = torch.stack([-b, a], dim=-2).flatten(-3)
    return x * cos + turned * sin


def _plain_append(s):
    norm = s["norm"] or (None,) * 4
    q = _plain_prologue(s["q"], norm[0], norm[1], s).to(s["q"].dtype)
    k = _plain_prologue(s["k"], norm[2], norm[3], s)
    b, t = k.shape[:2]
    lens = s["lens"].long()
    n_new = s["n_new"].long() if s["n_new"] is not None else torch.full_like(lens, t)
    touched = (t + PAGE - 2) // PAGE + 1  # pages that t tokens can reach into, wherever the first one falls
    page = torch.arange(touched, device=k.device)
    ids = torch.gather(s["table"].long(), 1, (lens // PAGE)[:, None] + page)
    # the new token that each slot of those pages takes, and the slots that hold one already
    token = page[:, None] * PAGE + torch.arange(PAGE, device=k.device) - (lens % PAGE)[:, None, None]
    fresh = (token >= 0) & (token < n_new[:, None, None])
    take = token.clamp(0, t - 1).flatten(1)
    stream = torch.arange(b, device=k.device)[:, None]
    for name, x in (("k", k), ("v", s["v"].float())):
        x = x[stream, take].unflatten(1, (touched, PAGE)).transpose(2, 3)  # (b, touched, heads, 64, 64)
        _plain_store(s[name + "_pages"], s[name + "_scale"], x, ids, fresh[:, :, None, :, None],
                     (token < 0)[:, :, None, :, None])
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _plain_store(pages, scale, x, ids, fresh, held):
    """Writes the fresh slots of the pages `ids`, at the scale that all of a page's tokens need."""
    x = torch.where(fresh, x, torch.zeros_like(x))
    codes, before = pages.view(torch.uint8)[ids], scale.view(torch.uint8)[ids].int()
    u = _scale_codes(x.abs().amax((-1, -2)))
    u = torch.where(held.any(-2)[..., 0], torch.maximum(u, before), u)
    u = torch.where(fresh.any(-2)[..., 0], u, before)
    # what a page held already moves to its new scale
    moved = codes.view(torch.float8_e4m3fn).float() * (_scale_values(before) * _scale_inverse(u))[..., None, None]
    new = (x * _scale_inverse(u)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    held = held & (u != before)[..., None, None]
    codes = torch.where(fresh, new, torch.where(held, moved.to(torch.float8_e4m3fn).view(torch.uint8), codes))
    pages.view(torch.uint8)[ids] = codes
    scale.view(torch.uint8)[ids] = u.to(torch.uint8)


def _plain_attend(s):
    q = s["q"].float()
    b, t, hq, _ = q.shape
    hkv = s["k_pages"].shape[1]
    table = s["table"].long()

    def tokens(name):  # (b, hkv, 1, tokens, 64)
        x = s[name + "_pages"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        x = x * _scale_values(s[name + "_scale"].view(torch.uint8)[table].int())[..., None, None]
        return x.transpose(1, 2).flatten(2, 3)[:, :, None]

    k = tokens("k")
    q = q.view(b, t, hkv, hq // hkv, HD).permute(0, 2, 3, 1, 4)
    score = (q * (1.0 / math.sqrt(HD))) @ k.transpose(-1, -2)  # (b, hkv, g, t, tokens)
    seen = s["lens"][:, None].expand(b, t)
    if s["limits"] is not None:
        seen = torch.minimum(seen, s["limits"])
    hidden = torch.arange(k.shape[-2], device=q.device) >= seen[:, None, None, :, None]
    score.masked_fill_(hidden, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ tokens("v")) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, hq, HD).to(s["q"].dtype)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)


def _exact_linear(s):
    x, w = s["x"].double(), s["w8"].double()
    out = torch.empty(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    step = max(1, (1 << 27) // max(w.shape))
    for at in range(0, x.shape[0], step):
        part = x[at:at + step]
        unit = part.abs().max(dim=-1).values / 127
        unit[unit == 0] = 1
        whole = torch.round(part / unit[:, None])
        y = torch.einsum("mk,nk->mn", whole, w) * unit[:, None] * s["w_scale"].double() + s["bias"].double()
        if s["act"] == "gelu":
            y = torch.special.ndtr(y) * y
        out[at:at + step] = y
    return out


def _exact_append(s):
    norm = [None if p is None else p.double() for p in (s["norm"] or (None,) * 4)]
    # the rotation as complex numbers: feature i of a half pairs with i + 16
    turn = torch.complex(s["cos"].double(), s["sin"].double())[:, :16]

    def prologue(x, weight, bias):
        x = x.double()
        if weight is not None:
            var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
            x = (x - mean) / (var + 1e-5).sqrt() * weight + bias
        parts = []
        for axis in range(2):
            half = x[..., 32 * axis:32 * axis + 32]
            z = torch.complex(half[..., :16], half[..., 16:]) * turn[s["pos"][..., axis]][:, :, None]
            parts += [z.real, z.imag]
        return torch.cat(parts, dim=-1)

    def e4m3(x):  # to the nearest, ties to even: 4 significant bits, steps of 2^-9 at least
        step = torch.exp2((torch.frexp(x.abs())[1] - 4).clamp(min=-9).double())
        return torch.round(x / step) * step

    q = prologue(s["q"], norm[0], norm[1])
    k, v = prologue(s["k"], norm[2], norm[3]), s["v"].double()
    lens = s["lens"].tolist()
    counts = s["n_new"].tolist() if s["n_new"] is not None else [k.shape[1]] * k.shape[0]
    table = s["table"].tolist()
    out = {}
    for name, x in (("k", k), ("v", v)):
        pages = s[name + "_pages"].view(torch.float8_e4m3fn).float()
        exponent = s[name + "_scale"].view(torch.uint8).long() - 127
        for b, (held, n) in enumerate(zip(lens, counts)):
            done = 0
            while done < n:
                where, slot = table[b][(held + done) // PAGE], (held + done) % PAGE
                take = min(PAGE - slot, n - done)
                fresh = x[b, done:done + take].transpose(0, 1)  # (heads, take, 64)
                # the least e with amax <= 448 * 2^e
                amax = fresh.abs().amax((-1, -2))
                e = torch.where(amax > 0, torch.ceil(torch.log2(amax / 448)), torch.full_like(amax, -127)).long()
                if slot:
                    old = exponent[where].clone()
                    e = torch.maximum(e, old)
                    back = pages[where, :, :slot].double() * torch.exp2((old - e).double())[:, None, None]
                    pages[where, :, :slot] = e4m3(back).float()
                pages[where, :, slot:slot + take] = e4m3(fresh / torch.exp2(e.double())[:, None, None]).float()
                exponent[where] = e
                done += take
        out[name] = pages, torch.exp2(exponent.double())
    return q, out["k"][0].double(), out["v"][0].double(), out["k"][1], out["v"][1]


def _exact_attend(s):
    q = s["q"].double()
    b, t, hq, _ = q.shape
    hkv = s["k_pages"].shape[1]
    out = torch.zeros(b, t, hq, HD, dtype=torch.float64, device=q.device)
    for i, held in enumerate(s["lens"].tolist()):
        ids = s["table"][i, :_pages(held)].long()
        for h in range(hkv):
            k, v = ((s[n + "_pages"].view(torch.uint8)[ids, h].view(torch.float8_e4m3fn).double()
                     * torch.exp2(s[n + "_scale"].view(torch.uint8)[ids, h].double() - 127)[:, None, None])
                    .reshape(-1, HD)[:held] for n in ("k", "v"))
            for head in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                score = torch.einsum("td,kd->tk", q[i, :, head], k) / HD ** 0.5
                if s["limits"] is not None:
                    score[torch.arange(held, device=q.device) >= s["limits"][i, :, None]] = -torch.inf
                # a row that sees nothing gives zeros
                out[i, :, head] = torch.nan_to_num(torch.softmax(score, dim=-1)) @ v
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        size = 2 if case["dtype"] == "bf16" else 4
        return dict(bytes=m * (k + n) * size + n * k + 8 * n, flops=2 * m * n * k)
    b, t, hq, hkv = case["b"], case["t"], case["hq"], case["hkv"]
    if case["op"] == "append":
        size = 2 if case["dtype"] == "bf16" else 4
        new = b * t * (0.5 if case["ragged"] else 1)
        # q, k and v read; q, and 8 bits each of k and v, written
        return dict(bytes=new * HD * (2 * hq * size + 2 * hkv * (size + 1)) + new * 16,
                    flops=new * HD * (hq + 2 * hkv) * (12 if case["norm"] else 6))
    held = case["held"] * (0.625 if case["ragged"] else 1)
    seen = held - (t - 1) / 2 if case["mask"] == "causal" else held
    if case["mask"] == "frame" and t > FRAME:
        seen = held - (t - FRAME) / 2
    return dict(bytes=b * (held * hkv * (2 * HD + 2 / PAGE) + 2 * t * hq * HD * 2), flops=4 * b * hq * t * HD * max(seen, 1))
