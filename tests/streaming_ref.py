"""64-bit references of the streaming operators, written from their formulas:
the paged e4m3 cache (append, attention) and the int8 Linear."""

import torch

PAGE, HD = 64, 64
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def make_cache(n_pages, heads, device="cuda", fill=0xFF):
    """Pages and scales whose every byte is `fill` (0xFF: NaN codes, NaN scales)."""
    def raw(*shape):
        return torch.full(shape, fill, dtype=torch.uint8, device=device)

    return dict(k_pages=raw(n_pages, heads, PAGE, HD).view(E4M3), v_pages=raw(n_pages, heads, PAGE, HD).view(E4M3),
                k_scale=raw(n_pages, heads).view(E8M0), v_scale=raw(n_pages, heads).view(E8M0))


def shuffled_table(streams, width, n_pages, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(n_pages, generator=g)[:streams * width].to(torch.int32).view(streams, width).to(device)


def norm_rotate(x, weight, bias, eps, pos, cos, sin):
    """(B, T, H, 64) -> LayerNorm over the head dims, then the 2-D rotation, in fp64."""
    x = x.double()
    if weight is not None:
        mean = x.mean(-1, keepdim=True)
        var = ((x - mean) ** 2).mean(-1, keepdim=True)
        x = (x - mean) / torch.sqrt(var + eps) * weight.double() + bias.double()
    if cos is not None:
        p = pos.clamp(0, cos.shape[0] - 1)
        c = torch.cat([cos.double()[p[..., 0]], cos.double()[p[..., 1]]], -1)[:, :, None]
        s = torch.cat([sin.double()[p[..., 0]], sin.double()[p[..., 1]]], -1)[:, :, None]
        h = x.reshape(*x.shape[:-1], 2, 2, 16)
        x = x * c + torch.stack([-h[..., 1, :], h[..., 0, :]], -2).reshape(x.shape) * s
    return x


def least_scale(amax):
    """e with amax <= 448 * 2^e, as small as possible (at least -127)."""
    e = -127
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def dense_kv(cache, table, lens, b, h):
    """Keys and values (fp64) of stream b's tokens, head h."""
    n = int(lens[b])
    ids = table[b, :-(-n // PAGE)].long()
    out = []
    for w in "kv":
        codes = cache[w + "_pages"].view(torch.uint8)[ids, h].view(E4M3).double()
        u = cache[w + "_scale"].view(torch.uint8)[ids, h].double()
        f = torch.where(u == 255, torch.full_like(u, torch.nan), torch.exp2(u - 127))
        out.append((codes * f[:, None, None]).reshape(-1, HD)[:n])
    return out


def attention(q, cache, table, lens, limits=None, sm_scale=0.125):
    """fp64 attention of q (B, T, Hq, 64) over the cache, and sum(p |v|): the
    size against which errors of P count.  Hidden tokens take no part at all."""
    B, T, Hq, _ = q.shape
    Hkv = cache["k_pages"].shape[1]
    ref = torch.zeros(B, T, Hq, HD, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(ref)
    for b in range(B):
        n = int(lens[b])
        for h in range(Hkv):
            k, v = dense_kv(cache, table, lens, b, h)
            for g in range(Hq // Hkv):
                hq = h * (Hq // Hkv) + g
                s = q[b, :, hq].double() @ k.t() * sm_scale
                seen = torch.full((T,), n, device=q.device) if limits is None else limits[b].clamp(0, n)
                hide = torch.arange(n, device=q.device)[None] >= seen[:, None]
                p = torch.softmax(s.masked_fill(hide, -torch.inf), -1) if n else s
                p = torch.where(hide, torch.zeros_like(p), p)
                p = torch.where((seen == 0)[:, None], torch.zeros_like(p), p)
                ref[b, :, hq], size[b, :, hq] = p @ v, p @ v.abs()
    return ref, size


def quant_rows(x):
    """Codes (fp64 integers) and fp32 scales, by the operator's fp32 steps."""
    x = x.float()
    scale = x.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)
    d = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(x / d[..., None]).double(), scale
