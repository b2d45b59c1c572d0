"""Views one after another: global attention over a growing 8-bit cache.

The reference's global attention takes all views of a scene at once.  Here a
model keeps, per global block, the keys and values of the frames it has seen
(pages of 64 tokens in e4m3 with one power-of-two scale per page and head: a
quarter of fp32, half of bf16), and each new frame attends to those before it
and to itself.  With ``quantize_linears`` its Linear layers run in 8-bit
integers as well.

    model = vggt.VGGTAggregatorModel().cuda().bfloat16().eval()
    stream.quantize_linears(model.aggregator.global_blocks)
    stream.apply_stream(model, streams=1, max_frames=200, frame_tokens=1374)
    for i, frame in enumerate(frames):                    # (1, 1, 3, H, W)
        out, _ = model(frame, first_frame=i == 0)
    stream.reset_stream(model)                            # the next scene
"""

from __future__ import annotations

from types import MethodType

import torch
import torch.nn as nn

from . import kernels as K
from ._lib import RessError
from .wiring import global_blocks


class StreamCache:
    """The keys and values of one attention layer, for several streams: a pool
    of pages, each stream's pages, and the tokens it holds."""

    def __init__(self, streams: int, heads: int, max_tokens: int, device="cuda"):
        self.pages_per_stream = -(-max_tokens // K.PAGE)
        n = streams * self.pages_per_stream
        if streams < 1 or heads < 1 or max_tokens < 1:
            raise RessError("a cache has streams, heads and tokens")
        self.max_tokens = max_tokens
        self.k_pages, self.v_pages = (torch.empty(n, heads, K.PAGE, K.HD, dtype=torch.float8_e4m3fn, device=device)
                                      for _ in range(2))
        self.k_scale, self.v_scale = (torch.empty(n, heads, dtype=torch.float8_e8m0fnu, device=device) for _ in range(2))
        self.table = torch.arange(n, dtype=torch.int32, device=device).view(streams, self.pages_per_stream)
        self.lens = torch.zeros(streams, dtype=torch.int32, device=device)
        self._most = 0  # tokens that the longest stream can hold by now

    @property
    def tensors(self) -> dict:
        """The cache's arguments of ``kernels.cache_append`` and ``cache_attn``."""
        return dict(k_pages=self.k_pages, v_pages=self.v_pages, k_scale=self.k_scale, v_scale=self.v_scale,
                    table=self.table, lens=self.lens)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tensors.values())

    def append(self, k, v, q=None, n_new=None, **prologue):
        """Adds k, v (streams, T, heads, 64) behind what the streams hold, the
        first n_new (streams,) of them where given; returns q's rows, normalised
        and rotated as k's (kernels.cache_append).  Whether they fit is known
        without a look at the device until the longest stream may be full,
        padding counted; from then on a call waits for the lengths."""
        T = k.shape[1]
        if n_new is not None and (not isinstance(n_new, torch.Tensor) or n_new.device != self.lens.device):
            raise RessError("n_new must be a tensor on the cache's device")
        new = T if n_new is None else n_new.clamp(0, T)  # as the call takes it
        most = self._most + T
        if most > self.max_tokens and not torch.cuda.is_current_stream_capturing():
            most = int((self.lens + new).max())
        if most > self.max_tokens:
            raise RessError(f"the cache holds {self.max_tokens} tokens a stream: with {T} more there may be {most}, which do "
                            "not fit")
        rows = K.cache_append(k, v, **self.tensors, q=q, n_new=n_new, **prologue)
        self.lens += new
        self._most = most
        return rows

    def attend(self, q, limits=None, **kw):
        """Attention of q (streams, T, heads, 64) over what the streams hold (kernels.cache_attn)."""
        return K.cache_attn(q, **self.tensors, limits=limits, **kw)

    def reset(self):
        """Forgets every stream's tokens."""
        self.lens.zero_()
        self._most = 0


class Int8Linear(nn.Module):
    """A Linear in 8-bit integers: one scale per output channel, laid out here,
    and one per token, found in the call (kernels.int8_linear)."""

    def __init__(self, linear: nn.Linear, act: str | None = None):
        super().__init__()
        self.in_features, self.out_features, self.act = linear.in_features, linear.out_features, act
        self.dtype = linear.weight.dtype
        w8, scale = K.int8_quant_rows(linear.weight.detach())
        self.register_buffer("w8", w8)
        self.register_buffer("scale", scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float())

    @property
    def weight(self) -> torch.Tensor:
        """The weight that the codes stand for, in the type of the Linear this was."""
        return (self.w8.float() * self.scale[:, None]).to(self.dtype)

    def forward(self, x):
        if not torch.is_autocast_enabled("cuda"):
            return K.int8_linear(x, self.w8, self.scale, self.bias, act=self.act)
        # as a Linear's, the output has autocast's type; fp16, which the kernel has not, goes by fp32
        dtype = torch.get_autocast_dtype("cuda")
        x = x.float() if x.dtype == torch.float16 else x
        out = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
        return K.int8_linear(x, self.w8, self.scale, self.bias, act=self.act, out_dtype=out).to(dtype)

    def _apply(self, fn, recurse=True):
        # .to(dtype), .half() and the like move the module and change the type it
        # stands for, but keep its scales and bias in fp32
        kept = {n: b for n, b in self._buffers.items() if b is not None and b.dtype == torch.float32}
        self.dtype = fn(torch.empty(0, dtype=self.dtype, device=self.w8.device)).dtype
        super()._apply(fn, recurse)
        for n, b in kept.items():
            self._buffers[n] = b.to(self._buffers[n].device)
        return self

    def extra_repr(self):
        return f"{self.in_features}, {self.out_features}, bias={self.bias is not None}, act={self.act}"


def quantize_linears(module: nn.Module) -> int:
    """Replaces every Linear below ``module`` whose width the kernel takes (a
    multiple of 16) by an Int8Linear; an MLP's first Linear takes its GELU
    along.  Returns how many."""
    from .vggt import Mlp

    n = 0
    for parent in list(module.modules()):
        for name, child in list(parent.named_children()):
            if type(child) is nn.Linear and child.in_features % 16 == 0:
                setattr(parent, name, Int8Linear(child, "gelu" if type(parent) is Mlp and name == "fc1" else None))
                n += 1
    return n


def _prologue(attn) -> dict:
    """The norms and rotary tables of a block, as cache_append takes them."""
    args = {}
    for name, norm in (("qn", attn.q_norm), ("kn", attn.k_norm)):
        if isinstance(norm, nn.Identity):
            continue
        if not isinstance(norm, nn.LayerNorm) or tuple(norm.normalized_shape) != (K.HD,) or norm.weight is None or \
                norm.bias is None:
            raise RessError("streaming takes q/k LayerNorms over 64 head dims, with weight and bias, or none")
        for part in ("weight", "bias"):
            p = getattr(norm, part).detach()
            args[f"{name}_{part}"] = p if p.dtype in (torch.float32, torch.bfloat16) else p.float()
        if args.setdefault("eps", norm.eps) != norm.eps:
            raise RessError("streaming takes q/k LayerNorms of one eps")
    rope = getattr(attn, "rope", None)
    if rope is not None:
        from .vggt import RotaryPosition2D

        if type(rope) is not RotaryPosition2D:
            raise RessError("streaming takes the 2-D table rotary embedding (vggt.RotaryPosition2D), or none")
    return args


def stream_attention_forward(attn, x, pos, cache: StreamCache, frame_tokens: int, prologue: dict):
    """A global block's attention on new frames x (streams, frames * frame_tokens,
    C): they join the cache, and each sees the frames up to its own."""
    B, T, C = x.shape
    H = attn.num_heads
    if T % frame_tokens:
        raise RessError(f"{T} tokens are no whole number of frames of {frame_tokens}")
    lin = attn.qkv(x).view(B, T, 3, H, C // H)
    kw = dict(prologue)
    if getattr(attn, "rope", None) is not None and pos is not None:
        cos, sin = attn.rope._cos_sin(K.HD // 2, attn.rope.MAX_POS, x.device, lin.dtype)
        kw.update(rope_cos=cos, rope_sin=sin, pos=pos.to(torch.int64))
    limits = None
    if T > frame_tokens:
        ends = (torch.arange(T, device=x.device, dtype=torch.int32) // frame_tokens + 1) * frame_tokens
        limits = (cache.lens[:, None] + ends).contiguous()
    q = cache.append(lin[:, :, 1], lin[:, :, 2], q=lin[:, :, 0], **kw)
    # fp32 queries are rounded to bf16, which the kernels take: 2^-8 of an element, beside the
    # 2^-4 of the keys' codes.  What comes out keeps the projection's type.
    o = cache.attend(q if q.dtype == torch.bfloat16 else q.bfloat16(), limits=limits,
                     out_bf16=lin.dtype == torch.bfloat16)
    return attn.proj_drop(attn.proj(o.view(B, T, C).to(x.dtype)))


def apply_stream(model, streams: int = 1, max_frames: int = 64, frame_tokens: int = 1374):
    """Installs streaming global attention: every call of the model brings new
    frames (``first_frame`` False after the first), which attend to the frames
    before them.  One cache per global block, for ``max_frames`` frames of
    ``frame_tokens`` tokens (special tokens included) in each of ``streams``
    batch rows.  ``remove_stream`` takes it out again."""
    remove_stream(model)
    for block in global_blocks(model):
        attn = block.attn
        p = next(attn.parameters(), None)
        device = p.device if p is not None else next(attn.buffers()).device
        cache = StreamCache(streams, attn.num_heads, max_frames * frame_tokens, device)
        _prologue(attn)  # refused here, not at the first frame

        def _fwd(self, x, pos=None, xpos=None, attn_bias=None, attn_mask=None, _cache=cache):
            if attn_bias is not None or attn_mask is not None:
                raise AssertionError("streaming attention decides what each frame sees; a caller-side attn_bias or "
                                     "attn_mask has no place in it")
            # the norms as they are now: weights may have been loaded or moved since
            return stream_attention_forward(self, x, pos if pos is not None else xpos, _cache, frame_tokens, _prologue(self))

        forward = MethodType(_fwd, attn)
        attn.ress_stream = (cache, attn.__dict__.get("forward"), forward)
        attn.forward = forward
    return model


def stream_caches(model) -> list:
    return [block.attn.ress_stream[0] for block in global_blocks(model)]


def reset_stream(model):
    """Forgets the frames seen: the next call starts a scene."""
    for cache in stream_caches(model):
        cache.reset()
    return model


def remove_stream(model):
    """Puts the global blocks' attention back to what it was before apply_stream;
    a forward that was installed over it since stays."""
    for block in global_blocks(model):
        state = block.attn.__dict__.pop("ress_stream", None)
        if state is not None and block.attn.__dict__.get("forward") is state[2]:
            del block.attn.forward
            if state[1] is not None:
                block.attn.forward = state[1]
    return model
