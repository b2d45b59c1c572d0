"""The streaming calls without a GPU: the C entries refuse bad arguments before
they touch a device, their structs have the layout the binding packs, the
64-bit references agree with torch's own casts, and a model is wired and
unwired."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch

from ress_b200 import _lib, stream, vggt
from ress_b200._lib import RessError

from streaming_ref import E4M3, PAGE, attention, least_scale, make_cache, quant_rows, shuffled_table

FAKE = 1 << 20  # never dereferenced: refused before any launch


def _cache(**kw):
    f = dict(k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, n=4, heads=2, ps=8192, hs=4096, ss=2, table=FAKE, ts=4, width=4, lens=FAKE,
             streams=1)
    f.update(kw)
    return _lib.CACHE.pack(*f.values())


def _append(**kw):
    f = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, dtype=1, tokens=3, q_heads=2, qsb=384, qst=128, qsh=64, ksb=384, kst=128,
             ksh=64, vsb=384, vst=128, vsh=64, qw=FAKE, qb=FAKE, kw=FAKE, kb=FAKE, eps=1e-5, pos=FAKE, cos=FAKE, sin=FAKE,
             rope=8, n_new=0)
    f.update(kw)
    return _lib.APPEND_ARGS.pack(*f.values())


def _attn(**kw):
    f = dict(q=FAKE, out=FAKE, tokens=3, q_heads=2, qsb=384, qst=128, qsh=64, osb=384, ost=128, osh=64, bf16=1, limits=0,
             scale=0.125, ws=0)
    f.update(kw)
    return _lib.ATTN_ARGS.pack(*f.values())


BAD_CACHE = [dict(k=0), dict(v=0), dict(ks=0), dict(vs=0), dict(table=0), dict(lens=0), dict(n=0), dict(heads=0),
             dict(streams=0), dict(width=0), dict(k=FAKE + 4), dict(ps=8200), dict(hs=4000), dict(ss=1)]


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_bad_caches_are_refused(kw):
    lib = _lib.load()
    assert lib.ress_cache_append(_cache(**kw), _append(), FAKE, None) == _lib.RESS_E_ARG
    assert lib.ress_cache_attn(_cache(**kw), _attn(), FAKE, None) == _lib.RESS_E_ARG


@pytest.mark.parametrize("kw,code", [
    (dict(k=0), -1), (dict(v=0), -1), (dict(tokens=0), -1), (dict(out=0), -1), (dict(q=0), -1), (dict(q_heads=3), -1),
    (dict(qb=0), -1), (dict(kw=0), -1), (dict(sin=0), -1), (dict(pos=0), -1), (dict(rope=0), -1), (dict(dtype=2), -2),
    (dict(k=FAKE + 2), -1), (dict(kst=130), -1), (dict(qsh=60), -1), (dict(kb=FAKE + 4), -1), (dict(tokens=1 << 23), -3)])
def test_bad_appends_are_refused(kw, code):
    assert _lib.load().ress_cache_append(_cache(), _append(**kw), FAKE, None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=0), -1), (dict(out=0), -1), (dict(tokens=0), -1), (dict(q_heads=3), -1), (dict(q=FAKE + 2), -1),
    (dict(qst=100), -1), (dict(ost=68, bf16=1), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1),
    (dict(tokens=1 << 31), -3), (dict(tokens=1 << 11, ws=0), -1)])
def test_bad_attention_calls_are_refused(kw, code):
    wide = _cache(width=64)  # long enough for the pages to be split, which needs a workspace
    assert _lib.load().ress_cache_attn(wide, _attn(**kw), FAKE, None) == code


def test_null_structs_and_status_are_refused():
    lib = _lib.load()
    assert lib.ress_cache_append(None, _append(), FAKE, None) == -1
    assert lib.ress_cache_append(_cache(), None, FAKE, None) == -1
    assert lib.ress_cache_append(_cache(), _append(), None, None) == -1
    assert lib.ress_cache_attn(_cache(), None, FAKE, None) == -1
    assert lib.ress_cache_attn(_cache(), _attn(), None, None) == -1


def test_structs_hold_eight_byte_fields():
    for packed in (_lib.CACHE, _lib.APPEND_ARGS, _lib.ATTN_ARGS):
        assert packed.size == 8 * len(packed.format)


def test_workspaces():
    lib = _lib.load()
    assert lib.ress_cache_attn_workspace(1, 16, 1, 700) == 0
    assert lib.ress_cache_attn_workspace(0, 16, 1000, 700) == 0
    assert lib.ress_cache_attn_workspace(1, 16, 1374, 172) > 0
    assert lib.ress_int8_linear_workspace(1, 1024) == 0
    assert lib.ress_int8_linear_workspace(1000, 1024) >= 1000 * 1024 + 4000
    assert lib.ress_int8_linear_workspace(0, 1024) == 0


@pytest.mark.parametrize("change,code", [
    (dict(x=0), -1), (dict(w=0), -1), (dict(scale=0), -1), (dict(out=0), -1), (dict(status=0), -1), (dict(M=0), -1),
    (dict(st=32), -1), (dict(ost=8), -1), (dict(dt=3), -2), (dict(odt=-1), -2), (dict(K=72, st=72), -3),
    (dict(x=FAKE + 2), -1), (dict(w=FAKE + 8), -1), (dict(st=65), -1), (dict(M=100, ws=0), -1), (dict(ws=FAKE + 4), -1)])
def test_bad_linears_are_refused(change, code):
    f = dict(x=FAKE, dt=1, M=4, N=16, K=64, st=64, w=FAKE, scale=FAKE, bias=FAKE, gelu=0, out=FAKE, odt=1, ost=16, ws=FAKE,
             status=FAKE, stream=0)
    f.update(change)
    ptr = {"x", "w", "scale", "bias", "out", "ws", "status", "stream"}
    args = [ctypes.c_void_p(v) if k in ptr else v for k, v in f.items()]
    assert _lib.load().ress_int8_linear(*args) == code


def test_bad_row_quantisers_are_refused():
    f = _lib.load().ress_int8_quant_rows
    p = ctypes.c_void_p(FAKE)
    assert f(None, 1, 1, 64, 64, p, p, None) == -1
    assert f(p, 1, 1, 64, 32, p, p, None) == -1
    assert f(p, 5, 1, 64, 64, p, p, None) == -2
    assert f(p, 1, 1, 24, 24, p, p, None) == -3
    assert f(ctypes.c_void_p(FAKE + 2), 1, 1, 64, 64, p, p, None) == -1


def test_references_agree_with_torch():
    """The references themselves: the least scale, and attention over a cache against plain softmax."""
    for amax in (1e-3, 0.4375, 0.44, 448.0, 449.0, 1e5):
        e = least_scale(amax)
        assert amax <= 448 * 2.0 ** e and amax > 448 * 2.0 ** (e - 1)
    g = torch.Generator().manual_seed(0)
    cache = make_cache(5, 1, device="cpu", fill=0)
    table = shuffled_table(1, 3, 5, seed=1, device="cpu")
    lens = torch.tensor([100])
    k, v = torch.randn(2, 100, 64, generator=g).to(E4M3).float()
    for name, x in (("k", k), ("v", v)):
        for i in range(100):
            cache[name + "_pages"][table[0, i // PAGE].long(), 0, i % PAGE] = x[i].to(E4M3)
        cache[name + "_scale"].view(torch.uint8).fill_(127 + 2)
    q = torch.randn(1, 2, 1, 64, generator=g)
    ref, size = attention(q, cache, table, lens)
    want = torch.softmax(q[0, :, 0].double() @ (4 * k.double()).t() / 8, -1) @ (4 * v.double())
    assert torch.allclose(ref[0, :, 0], want, atol=1e-12) and bool((size >= ref.abs()).all())
    x8, s = quant_rows(torch.tensor([[1.0, -127.0, 3.4], [0.0, 0.0, 0.0]]))
    assert x8.tolist() == [[1, -127, 3], [0, 0, 0]] and s[1] == 0


def test_wiring_without_a_gpu():
    m = vggt.VGGTAggregatorModel(dim=128, depth=2, num_heads=2, img=28, encoder_depth=1)
    stream.apply_stream(m, streams=2, max_frames=3, frame_tokens=9)
    caches = stream.stream_caches(m)
    assert len(caches) == 2 and caches[0].table.shape == (2, 1) and caches[0].k_pages.shape == (2, 2, 64, 64)
    x = torch.zeros(2, 9, 128)
    with pytest.raises(RessError, match="CUDA"):
        m.aggregator.global_blocks[0].attn(x, pos=torch.zeros(2, 9, 2, dtype=torch.long))
    with pytest.raises(AssertionError):
        m.aggregator.global_blocks[0].attn(x, attn_mask=x)
    stream.remove_stream(m)
    assert "forward" not in m.aggregator.global_blocks[0].attn.__dict__
    with pytest.raises(RessError):
        stream.quantize_linears(m)  # laid out on the GPU


# Two devices that do nothing: what the tensor library asks the runtime before a call.
FAKE_RUNTIME = """
static int device;
int cudaGetDeviceCount(int *n) { *n = 2; return 0; }
int cudaGetDevice(int *d) { *d = device; return 0; }
int cudaSetDevice(int d) { device = d; return 0; }
int cudaDeviceGetStreamPriorityRange(int *lo, int *hi) { *lo = 0; *hi = -5; return 0; }
"""
ON_ANOTHER_DEVICE = """
import ctypes, os, sys
import torch
from ress_b200 import _lib

class Meta(torch.Tensor):  # a tensor of device 1 without memory
    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        raise AssertionError(f)

def t(*shape, dtype=torch.float32):
    return torch.Tensor._make_wrapper_subclass(Meta, shape, dtype=dtype, device=torch.device("cuda", 1))

runtime = ctypes.CDLL(sys.argv[1])
def current():
    d = ctypes.c_int()
    runtime.cudaGetDevice(ctypes.byref(d))
    return d.value

# what the tensor library's own start-up would tell its device guard
has_context = ctypes.CFUNCTYPE(ctypes.c_bool, ctypes.c_byte)(lambda i: True)
c10 = ctypes.CDLL(os.path.join(os.path.dirname(torch.__file__), "lib", "libc10_cuda.so"))
c10._ZN3c104cuda9_internal20setHasPrimaryContextEPFbaE(has_context)

# entry points that note the current device
seen, P = [], ctypes.c_void_p
call = ctypes.CFUNCTYPE(ctypes.c_int, P, P, P, P)(lambda *a: (seen.append(current()), 0)[1])
size = ctypes.CFUNCTYPE(ctypes.c_size_t, P, P, P, P)(lambda *a: 0)
names = dict.fromkeys(_lib.SIGNATURES, ctypes.cast(call, P).value)
names["ress_cache_attn_workspace"] = ctypes.cast(size, P).value
import importlib.util
spec = importlib.util.spec_from_file_location("ress_b200._host", _lib.HOST_PATH)
host = importlib.util.module_from_spec(spec)
spec.loader.exec_module(host)
word = ctypes.c_int()
host.bind(_lib.RessError, lambda i: ctypes.addressof(word), names)

pages, scales, ints = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.int32
cache = [t(4, 2, 64, 64, dtype=pages)] * 2 + [t(4, 2, dtype=scales)] * 2 + [t(1, 4, dtype=ints), t(1, dtype=ints)]
k, q = t(1, 3, 2, 64), t(1, 3, 2, 64, dtype=torch.bfloat16)
host.cache_append(k, k, *cache, *[None] * 6, 1e-5, None, None, None)
host.cache_attn(q, *cache, None, None, t(1, 3, 2, 64), True)
print(*seen, current())
"""


def test_calls_run_on_their_tensors_device(tmp_path):
    """Tensors of device 1 while device 0 is current: the entry points find device 1 current, and
    afterwards device 0 is again.  The runtime is a stand-in, nothing is launched."""
    source, library = tmp_path / "runtime.c", tmp_path / "runtime.so"
    source.write_text(FAKE_RUNTIME)
    subprocess.run(["cc", "-shared", "-fPIC", str(source), "-o", str(library)], check=True)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", ON_ANOTHER_DEVICE, str(library)], capture_output=True, text=True, cwd=root,
                       env={**os.environ, "LD_PRELOAD": str(library), "PYTHONPATH": root})
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["1", "1", "0"]


@pytest.mark.parametrize("heads", [32768, 65535])
def test_heads_beyond_a_grid_are_refused(heads):
    """Two tiles of rows a head make more blocks than a grid's second dimension takes."""
    wide = _cache(heads=heads, ps=heads * 4096, ss=heads)
    assert _lib.load().ress_cache_attn(wide, _attn(tokens=20, q_heads=heads), FAKE, None) == -3


def test_norms_of_unlike_eps_are_refused():
    attn = vggt.Attention(128, 2, True, vggt.RotaryPosition2D())
    attn.k_norm.eps = 1e-3
    with pytest.raises(RessError, match="eps"):
        stream._prologue(attn)
    attn.q_norm.eps = 1e-3
    assert stream._prologue(attn)["eps"] == 1e-3
    attn.q_norm = torch.nn.Identity()
    attn.k_norm.eps = 1e-4
    assert stream._prologue(attn)["eps"] == 1e-4
