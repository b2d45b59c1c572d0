"""Streaming global attention (ress_b200.stream) on the VGGT-shaped aggregator:
frames fed one by one against the same model with exact frame-causal attention
in fp32, and the 8-bit Linears in it.

Tolerances: e4m3 keys and values err by 2^-4 of a value at most, 2 to 3 % of
its typical size on average, independently from token to token; an attention
output, an average over tokens, errs by about as much of its own size.  The
module test allows 5 % in the 2-norm and the model's outputs (the residual
stream, to which a block adds a hundredth) 2 % of the largest value, as the
other whole-model tests do.  int8 codes err by 1/254 of a row's largest
value."""

import pytest
import torch
import torch.nn.functional as F

from ress_b200 import kernels as K
from ress_b200 import stream, vggt
from ress_b200._lib import RessError

pytestmark = pytest.mark.gpu

IMG, FRAME = 112, 64 + 5


def _model(dtype=torch.bfloat16):
    torch.manual_seed(0)
    m = vggt.VGGTAggregatorModel(dim=256, depth=2, num_heads=4, img=IMG, encoder_depth=1, intermediate=(0, 1))
    return m.cuda().to(dtype).eval()


def _images(streams, frames):
    return torch.rand(streams, frames, 3, IMG, IMG, device="cuda", generator=torch.Generator("cuda").manual_seed(1))


def _frame_causal(attn, x, pos):
    """The attention module in fp32 with an exact frame-causal mask."""
    B, T, C = x.shape
    H = attn.num_heads
    q, k, v = attn.qkv(x).view(B, T, 3, H, C // H).permute(2, 0, 3, 1, 4).unbind(0)
    q, k = attn.rope(attn.q_norm(q), pos), attn.rope(attn.k_norm(k), pos)
    f = torch.arange(T, device=x.device) // FRAME
    o = F.scaled_dot_product_attention(q, k, v, attn_mask=f[:, None] >= f[None])
    return attn.proj(o.transpose(1, 2).reshape(B, T, C))


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("streams,chunks", [(1, [1] * 5), (2, [1, 3, 1]), (1, [5])])
def test_stream_matches_frame_causal_attention(streams, chunks):
    ref_model, m = _model(torch.float32), _model()
    images = _images(streams, 5)
    for block in ref_model.aggregator.global_blocks:
        block.attn.forward = lambda x, pos=None, _a=block.attn: _frame_causal(_a, x, pos)
    stream.apply_stream(m, streams=streams, max_frames=5, frame_tokens=FRAME)
    with torch.inference_mode():
        ref, _ = ref_model(images)
        got, at = [], 0
        for n in chunks:
            got.append(m(images[:, at:at + n], first_frame=at == 0)[0])
            at += n
    torch.cuda.synchronize()
    assert K.check_status() == 0
    for layer in range(2):
        out = torch.cat([g[layer] for g in got], 1).float()
        assert (out - ref[layer]).abs().max() <= 2e-2 * ref[layer].abs().max()
    assert stream.stream_caches(m)[0].lens.tolist() == [5 * FRAME] * streams


def test_stream_attention_module():
    torch.manual_seed(2)
    attn = vggt.Attention(256, 4, True, vggt.RotaryPosition2D()).cuda()
    x = torch.randn(2, 3 * FRAME, 256, device="cuda")
    pos = torch.randint(0, 9, (2, 3 * FRAME, 2), device="cuda")
    with torch.inference_mode():
        ref = _frame_causal(attn, x, pos)
        for dtype in (torch.float32, torch.bfloat16):
            a = attn.to(dtype)
            cache, pro = stream.StreamCache(2, 4, 3 * FRAME), stream._prologue(a)
            one = [stream.stream_attention_forward(a, x[:, i:i + FRAME].to(dtype), pos[:, i:i + FRAME], cache, FRAME, pro)
                   for i in range(0, 3 * FRAME, FRAME)]
            cache.reset()
            whole = stream.stream_attention_forward(a, x.to(dtype), pos, cache, FRAME, pro)
            assert whole.dtype == dtype
            assert _rel(torch.cat(one, 1), ref) < 0.05 and _rel(whole, ref) < 0.05
    assert K.check_status() == 0


def test_int8_linears_in_a_stream():
    m, q = _model(), _model()
    n = stream.quantize_linears(q.aggregator.frame_blocks) + stream.quantize_linears(q.aggregator.global_blocks)
    assert n == 4 * 4  # qkv, proj, fc1, fc2 of four blocks
    images = _images(1, 3)
    outs = []
    for model in (m, q):
        stream.apply_stream(model, max_frames=3, frame_tokens=FRAME)
        with torch.inference_mode():
            outs.append([model(images[:, i:i + 1], first_frame=i == 0)[0] for i in range(3)])
    torch.cuda.synchronize()
    assert K.check_status() == 0
    for a, b in zip(*outs):
        for x, y in zip(a, b):
            assert (x.float() - y.float()).abs().max() <= 2e-2 * x.float().abs().max()


def test_int8_linear_module():
    torch.manual_seed(3)
    lin = torch.nn.Linear(256, 96).cuda()
    x = torch.randn(4, 50, 256, device="cuda")
    q = stream.Int8Linear(lin)
    assert _rel(q(x), lin(x)) < 0.02
    assert _rel(stream.Int8Linear(lin, "gelu")(x), F.gelu(lin(x))) < 0.02
    b = stream.Int8Linear(torch.nn.Linear(256, 96, bias=False).cuda()).bfloat16()
    assert b.scale.dtype == torch.float32 and b.w8.dtype == torch.int8 and b(x.bfloat16()).dtype == torch.bfloat16
    assert (q.weight - lin.weight).abs().max() <= lin.weight.abs().max() / 254 * 1.01
    mlp = vggt.Mlp(64).cuda()
    y = torch.randn(30, 64, device="cuda")
    ref = mlp(y)
    assert stream.quantize_linears(mlp) == 2 and mlp.fc1.act == "gelu" and mlp.fc2.act is None
    assert _rel(mlp(y), ref) < 0.03


def test_reset_remove_and_refusals():
    m = _model()
    images = _images(1, 2)
    before = [b.attn.forward for b in m.aggregator.global_blocks]
    with torch.inference_mode():
        ref = m(images)[0]
        stream.apply_stream(m, max_frames=2, frame_tokens=FRAME)
        first = m(images[:, :1])[0]
        m(images[:, 1:], first_frame=False)
        with pytest.raises(RessError, match="do not fit"):
            m(images[:, :1], first_frame=False)
        stream.reset_stream(m)
        again = m(images[:, :1])[0]
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        with pytest.raises(RessError, match="whole number of frames"):
            stream.stream_attention_forward(m.aggregator.global_blocks[0].attn,
                                            torch.zeros(1, FRAME + 1, 256, device="cuda").bfloat16(), None,
                                            stream.stream_caches(m)[0], FRAME, {})
        stream.remove_stream(m)
        assert all(torch.equal(a, b) for a, b in zip(m(images)[0], ref))
    assert [b.attn.forward for b in m.aggregator.global_blocks] == before
    with pytest.raises(RessError):
        stream.StreamCache(1, 0, 10)
    odd = vggt.Attention(96, 3, True, None)  # 32 head dims
    with pytest.raises(RessError, match="64 head dims"):
        stream._prologue(odd)


def _cache_of(streams, tokens, heads=2):
    """A cache whose unused slots hold bytes that are no values."""
    c = stream.StreamCache(streams, heads, tokens)
    for t in (c.k_pages, c.v_pages, c.k_scale, c.v_scale):
        t.view(torch.uint8).fill_(0xFF)
    return c


@pytest.mark.parametrize("asked", [9, -3])
def test_cache_counts_what_was_stored(asked):
    """n_new beyond the tokens given, or below none: the lengths follow what the pages got."""
    g = torch.Generator("cuda").manual_seed(5)
    k, v = torch.randn(2, 2, 5, 2, 64, device="cuda", generator=g)
    c = _cache_of(2, 200)
    c.append(k, v)
    c.append(k, v, n_new=torch.tensor([asked, 2], dtype=torch.int32, device="cuda"))
    assert c.lens.tolist() == [5 + min(max(asked, 0), 5), 7]
    out = c.attend(torch.randn(2, 1, 2, 64, device="cuda", generator=g).bfloat16())
    assert bool(out.isfinite().all()) and K.check_status() == 0


def test_cache_counts_tokens_not_padding():
    """Padded appends whose tokens fit are taken; one that does not fit is not, and changes nothing."""
    g = torch.Generator("cuda").manual_seed(6)
    k, v = torch.randn(2, 3, 8, 2, 64, device="cuda", generator=g)
    c = _cache_of(3, 70)
    n_new = torch.tensor([1, 5, 0], dtype=torch.int32, device="cuda")
    for _ in range(14):  # 14 x 8 padded tokens, 70 in the longest stream
        c.append(k, v, n_new=n_new)
    assert c.lens.tolist() == [14, 70, 0]
    with pytest.raises(RessError, match="do not fit"):
        c.append(k, v, n_new=n_new)
    assert c.lens.tolist() == [14, 70, 0]
    c.append(k, v, n_new=torch.tensor([8, 0, 8], dtype=torch.int32, device="cuda"))
    assert c.lens.tolist() == [22, 70, 8]
    out = c.attend(torch.randn(3, 1, 2, 64, device="cuda", generator=g).bfloat16())
    assert bool(out.isfinite().all()) and K.check_status() == 0
    c.reset()
    c.append(k, v)
    assert c.lens.tolist() == [8, 8, 8]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_loaded_after_apply_stream(dtype):
    """The norms in use are the model's present ones, whatever its type."""
    m, fresh = _model(dtype), _model(dtype)
    state = {n: (t * (1 + 0.5 * torch.sin(torch.arange(t.numel(), device="cuda")).view_as(t))).to(t.dtype)
             if "_norm" in n else t for n, t in m.state_dict().items()}
    images = _images(1, 2)
    stream.apply_stream(m, max_frames=2, frame_tokens=FRAME)
    m.load_state_dict(state)
    fresh.load_state_dict(state)
    stream.apply_stream(fresh, max_frames=2, frame_tokens=FRAME)
    with torch.inference_mode():
        for i in range(2):
            a, b = (x(images[:, i:i + 1], first_frame=i == 0)[0] for x in (m, fresh))
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    # and they matter
    stream.reset_stream(m)
    other = stream.apply_stream(_model(dtype), max_frames=2, frame_tokens=FRAME)
    with torch.inference_mode():
        assert not torch.equal(m(images[:, :1])[0][0], other(images[:, :1])[0][0])


def test_int8_linears_on_the_sparse_path(monkeypatch):
    """The sparse path asks a quantised block for its type, not for its weights laid out again."""
    from ress_b200 import qkv

    torch.manual_seed(9)
    attn = vggt.Attention(256, 4, True, vggt.RotaryPosition2D()).cuda().bfloat16()
    stream.quantize_linears(attn)

    def unwanted(self):
        raise AssertionError("the weights were laid out")

    monkeypatch.setattr(stream.Int8Linear, "weight", property(unwanted))
    x = torch.randn(1, 2 * FRAME, 256, device="cuda").bfloat16()
    pos = torch.zeros(1, 2 * FRAME, 2, dtype=torch.long, device="cuda")
    with torch.inference_mode():
        assert qkv.compute_qkv_scored(attn, x, pos, 5, 4, shape=dict(H=8, W=8, N=2)) is not None
        qkv.project_out(attn, torch.randn(1, 4, 2 * FRAME, 64, device="cuda"), 1, 2, FRAME, 4, 64)


def test_int8_linear_type_follows_the_model():
    """Quantised in fp32 and then moved to bf16, a block is as one quantised from bf16 weights: type, and the sparse path's route."""
    from ress_b200 import qkv

    torch.manual_seed(8)
    attn = vggt.Attention(256, 4, True, vggt.RotaryPosition2D()).cuda()
    assert stream.quantize_linears(attn) == 2
    attn = attn.bfloat16()
    assert attn.qkv.dtype == torch.bfloat16 and attn.qkv.weight.dtype == torch.bfloat16
    assert attn.qkv.scale.dtype == torch.float32 and attn.qkv.bias.dtype == torch.float32
    x = torch.randn(1, 2 * FRAME, 256, device="cuda").bfloat16()
    pos = torch.zeros(1, 2 * FRAME, 2, dtype=torch.long, device="cuda")
    with torch.inference_mode():
        got = qkv.compute_qkv_scored(attn, x, pos, 5, 4, shape=dict(H=8, W=8, N=2))
        assert got is not None
        out = qkv.project_out(attn, torch.randn(1, 4, 2 * FRAME, 64, device="cuda"), 1, 2, FRAME, 4, 64)
    assert out.dtype == torch.bfloat16


def test_int8_linear_under_autocast():
    """As a Linear's, the output has autocast's type."""
    torch.manual_seed(10)
    lin = torch.nn.Linear(64, 32).cuda()
    q, x = stream.Int8Linear(lin), torch.randn(5, 64, device="cuda")
    with torch.inference_mode():
        assert q(x).dtype == torch.float32
        for dtype in (torch.bfloat16, torch.float16):
            with torch.autocast("cuda", dtype=dtype):
                assert q(x).dtype == lin(x).dtype == dtype
                assert _rel(q(x), lin(x)) < 0.02
                assert q(x.bfloat16()).dtype == q(x.to(dtype)).dtype == dtype


def test_remove_stream_leaves_what_came_later():
    m = _model()
    blocks = m.aggregator.global_blocks
    stream.apply_stream(m, max_frames=2, frame_tokens=FRAME)
    later = lambda x, pos=None: x  # noqa: E731
    blocks[0].attn.forward = later
    stream.remove_stream(m)
    assert blocks[0].attn.forward is later and "forward" not in blocks[1].attn.__dict__
    # taken out from between: what lies below is put back once
    blocks[0].attn.__dict__.pop("forward")
    blocks[1].attn.forward = later
    stream.apply_stream(m, max_frames=2, frame_tokens=FRAME)
    stream.apply_stream(m, max_frames=1, frame_tokens=FRAME)
    stream.remove_stream(m)
    assert "forward" not in blocks[0].attn.__dict__ and blocks[1].attn.forward is later


def test_fp32_streams_are_not_rounded_to_bf16():
    """The attention of an fp32 block comes out in fp32."""
    torch.manual_seed(7)
    attn = vggt.Attention(256, 4, True, vggt.RotaryPosition2D()).cuda()
    attn.proj = torch.nn.Identity()
    x, pos = torch.randn(1, FRAME, 256, device="cuda"), torch.randint(0, 9, (1, FRAME, 2), device="cuda")
    with torch.inference_mode():
        cache = stream.StreamCache(1, 4, FRAME)
        out = stream.stream_attention_forward(attn, x, pos, cache, FRAME, stream._prologue(attn))
    assert out.dtype == torch.float32
    assert (out != out.bfloat16().float()).float().mean() > 0.9


def test_inputs_that_need_gradients_are_refused():
    """The operators have no backward: no result without history for an input that has one."""
    x = torch.randn(1, 3, 2, 64, device="cuda", requires_grad=True)
    flat = torch.randn(4, 64, device="cuda", requires_grad=True)
    c = stream.StreamCache(1, 2, 64)
    w8, s = K.int8_quant_rows(torch.randn(8, 64, device="cuda"))
    q = x.detach().bfloat16().requires_grad_()
    plain = x.detach()
    weight = torch.ones(64, device="cuda", requires_grad=True)
    calls = [lambda: c.append(x, plain), lambda: c.append(plain, x), lambda: c.append(plain, plain, q=x), lambda: c.attend(q),
             lambda: c.append(plain, plain, kn_weight=weight, kn_bias=weight.detach()),
             lambda: K.int8_linear(flat, w8, s), lambda: K.int8_linear(flat.detach(), w8, s, weight[:8]),
             lambda: K.int8_quant_rows(flat)]
    for f in calls:
        with pytest.raises(RessError, match="no_grad"):
            f()
    with torch.no_grad():
        for f in calls:
            f()
    assert K.check_status() == 0
