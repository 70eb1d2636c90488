"""rope, kv_append_paged and attn_paged: what they refuse, by name and before any launch; and the host's part of rope. No GPU: the
runtime handle is one that a test built around the library's own struct, and every call ends in the checks."""
import ctypes as C
import subprocess
from dataclasses import replace
from pathlib import Path

import numpy as np
import pytest

from tessl_b200 import build, capi, nn

try:
    capi.load()
except ImportError:
    pytest.skip("the library is not built", allow_module_level=True)

CSRC = Path(build.__file__).parent / "csrc"
MAKE = """
#include "runtime.h"
extern "C" __attribute__((visibility("default"))) TesslRuntime *make()
{
    auto *rt = new TesslRuntime;
    rt->owner = std::this_thread::get_id(), rt->encode_only = true;
    return rt;
}
"""


class Handle:
    def __init__(self, p):
        self.handle = C.c_void_p(p)


@pytest.fixture(scope="module")
def host_rt(tmp_path_factory):
    d = tmp_path_factory.mktemp("host_rt")
    (d / "make.cpp").write_text(MAKE)
    cmd = ["g++", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), "-I", "/usr/local/cuda/include", "-o", str(d / "make.so"), str(d / "make.cpp")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        pytest.skip("no compiler with the CUDA headers: " + r.stderr[-200:])
    lib = C.CDLL(str(d / "make.so"))
    lib.make.restype = C.c_void_p
    return Handle(lib.make())


def refused(match, fn, *args, **kw):
    with pytest.raises(nn.TesslError, match=match) as e:
        fn(*args, **kw)
    assert e.value.status == capi.TESSL_ERR


at = iter(range(1 << 20, 1 << 40, 1 << 28))


def buf(nbytes, off=0):
    """A buffer that is never touched, far from the others."""
    return nn.GpuBuffer(next(at) + off, nbytes)


def null():
    return nn.GpuBuffer(0, 0)


# ------------------------------------------------------------------ rope ---

def rope_args(tokens=3, heads=2, dim=64, rot=64):
    plan = nn.Rope(buf(rot // 2 * 8), rot, False, 1.0)
    return dict(x=buf(tokens * heads * dim * 4), positions=buf(tokens * 4), out=buf(tokens * heads * dim * 2), rope=plan, tokens=tokens,
                n_heads=heads, head_dim=dim, x_as_bf16=False, out_as_bf16=True)


def call_rope(rt, **a):
    nn.rope(rt, **a)


@pytest.mark.parametrize("change,match", [
    (dict(head_dim=0), "head_dim 0"), (dict(head_dim=63), "head_dim 63"), (dict(head_dim=258), "head_dim 258"),
    (dict(head_dim=32), "rot_dim 64"), (dict(tokens=4), "positions|x"), (dict(n_heads=3), "rope x"), (dict(n_heads=1 << 21), "too many heads"),
    (dict(tokens=1 << 31), "too many tokens"), (dict(x_stride=100), "128 values long but 100 apart"), (dict(out_stride=4000), "rope out"),
])
def test_rope_refuses(host_rt, change, match):
    refused(match, call_rope, host_rt, **{**rope_args(), **change})


def test_rope_refuses_its_plan_and_places(host_rt):
    a = rope_args()
    refused("rot_dim 63", call_rope, host_rt, **{**a, "rope": replace(a["rope"], rot_dim=63)})
    refused("rope steps", call_rope, host_rt, **{**a, "rope": replace(a["rope"], steps=buf(31 * 8))})
    refused("8-byte aligned", call_rope, host_rt, **{**a, "rope": replace(a["rope"], steps=buf(1024, 4))})
    for f in (float("nan"), float("inf")):
        refused("not finite", call_rope, host_rt, **{**a, "rope": replace(a["rope"], factor=f)})
    refused("positions must be", call_rope, host_rt, **{**a, "positions": buf(64, 2)})
    refused("x is not aligned", call_rope, host_rt, **{**a, "x": buf(1 << 20, 2)})
    refused("overlaps read-only buffer x", call_rope, host_rt, **{**a, "out": nn.GpuBuffer(a["x"].ptr, a["out"].nbytes)})  # in place, but of another type
    refused("overlaps read-only buffer positions", call_rope, host_rt, **{**a, "out": nn.GpuBuffer(a["positions"].ptr, a["out"].nbytes)})
    refused("overlaps read-only buffer rope steps", call_rope, host_rt, **{**a, "out": nn.GpuBuffer(a["rope"].steps.ptr, a["out"].nbytes)})


def test_rope_of_nothing_is_done_at_once(host_rt):
    for z in (dict(tokens=0), dict(n_heads=0)):
        call_rope(host_rt, **{**rope_args(), **z})


# ----------------------------------------------------------------- steps ---

@pytest.mark.parametrize("rot", [0, 2, 64, 128, 256])
@pytest.mark.parametrize("theta", [10000.0, 1e6, 1.5])
def test_steps_are_the_frequencies(rot, theta):
    steps, factor = nn.rope_steps(rot, theta)
    assert factor == 1.0 and len(steps) == rot // 2
    w = theta ** (-2.0 * np.arange(rot // 2) / max(rot, 1)) / (2 * np.pi)
    # 2^64 w to the relative accuracy of the f64 on this side (power, quotient: a few 2^-53), and half a step
    assert (np.abs(np.asarray(steps, np.float64) - w * 2.0 ** 64) <= w * 2.0 ** 64 * 64 * 2.0 ** -53 + 1).all()


def test_scaled_steps_keep_order_and_bounds():
    plain = np.asarray(nn.rope_steps(128, 10000.0)[0], np.float64)
    for s in (nn.RopeScaling("linear", 4.0), nn.RopeScaling("ntk", 4.0), nn.RopeScaling("wavelength", 8.0, 8192.0),
              nn.RopeScaling("yarn", 4.0, 4096.0)):
        steps, factor = nn.rope_steps(128, 10000.0, s)
        got = np.asarray(steps, np.float64)
        assert (np.diff(got) < 0).all()
        assert (got <= plain * (1 + 2.0 ** -40)).all() and (got >= plain / s.factor * (1 - 2.0 ** -40) - 1).all()
        # 0.1 ln 4 + 1 in f32
        assert factor == (np.float32(0.1 * np.log(4.0) + 1.0) if s.kind == "yarn" else 1.0)
    one = nn.rope_steps(128, 10000.0, nn.RopeScaling("linear", 1.0))[0]
    assert np.array_equal(np.asarray(one, np.float64), plain)


@pytest.mark.parametrize("rot,theta,scaling,match", [
    (3, 1e4, None, "rot_dim 3"), (258, 1e4, None, "rot_dim 258"), (64, 1.0, None, "theta"), (64, float("nan"), None, "theta"),
    (64, float("inf"), None, "theta"), (64, 1e4, nn.RopeScaling("linear", 0.5), "factor"), (64, 1e4, nn.RopeScaling("ntk", float("inf")), "factor"),
    (64, 1e4, nn.RopeScaling("yarn", 2.0), "trained context"), (64, 1e4, nn.RopeScaling("wavelength", 2.0, -1.0), "trained context"),
    (64, 1e4, nn.RopeScaling("yarn", 2.0, 4096.0, 32.0, 1.0), "ascending"), (64, 1e4, nn.RopeScaling("wavelength", 2.0, 4096.0, -1.0, 4.0), "ascending"),
])
def test_steps_refuse(rot, theta, scaling, match):
    refused(match, nn.rope_steps, rot, theta, scaling)


# ------------------------------------------------- cache and sequences, both ---

def paged(n=3, new=(1, 1, 1), starts=False, pages=8, page=16, kvh=2, dim=64, width=4, **cache):
    total = sum(new)
    c = nn.PagedKv(buf(pages * page * kvh * dim * 2), buf(pages * page * kvh * dim * 2), pages, page, kvh, dim)
    s = nn.PagedSeqs(buf(n * width * 4), buf(n * 4), buf((n + 1) * 4) if starts else None, n, width)
    return replace(c, **cache), s, total


def call_attn(rt, cache, seqs, total, heads=4, q=None, out=None, work=None, **how):
    q, out = q or buf(total * heads * 256 * 2), out or buf(total * heads * 256 * 2)
    nn.attn_paged(rt, q, cache, seqs, out, work or buf(1 << 27), total, heads, how.pop("scale", 0.125), **how)


def call_append(rt, cache, seqs, total, heads=4, elem=4, **a):
    d, e = cache.head_dim, cache.n_kv_heads
    b = dict(q=buf(max(total, 1) * heads * max(d, 1) * elem), k=buf(max(total, 1) * e * max(d, 1) * elem), v=buf(max(total, 1) * e * max(d, 1) * elem),
             q_out=buf(max(total, 1) * heads * max(d, 1) * 2), rope=None, norm=None)
    b.update(a)
    nn.kv_append_paged(rt, b.pop("q"), b.pop("k"), b.pop("v"), b.pop("q_out"), cache, seqs, b.pop("rope"), b.pop("norm"), total, heads, in_as_bf16=elem == 2, **b)


CACHES = [(dict(layout=2), "layout 2"), (dict(head_dim=0), "head_dim 0"), (dict(head_dim=60), "head_dim 60"), (dict(head_dim=264), "head_dim 264"),
          (dict(n_kv_heads=0), "n_kv_heads 0"), (dict(n_kv_heads=65536), "n_kv_heads 65536"), (dict(page_size=0), "page_size"),
          (dict(page_size=1 << 25), "too large"), (dict(num_pages=1 << 31), "page id"), (dict(num_pages=9), "cache k"),
          (dict(k=nn.GpuBuffer(1 << 50, 1 << 20), v=null()), "cache v"), (dict(k=nn.GpuBuffer((1 << 50) + 8, 1 << 20)), "aligned")]


@pytest.mark.parametrize("call", [call_attn, call_append])
@pytest.mark.parametrize("change,match", CACHES)
def test_caches_that_are_refused(host_rt, call, change, match):
    cache, seqs, total = paged()
    refused(match, call, host_rt, replace(cache, **change), seqs, total)


@pytest.mark.parametrize("call", [call_attn, call_append])
def test_sequences_that_are_refused(host_rt, call):
    cache, seqs, total = paged()
    refused("each has one|each sequence has one", call, host_rt, cache, seqs, total + 1)
    refused("page_table", call, host_rt, cache, replace(seqs, max_pages=5), total)
    refused("page_table", call, host_rt, cache, replace(seqs, page_table=null()), total)
    refused("kv_lens", call, host_rt, cache, replace(seqs, kv_lens=buf(8)), total)
    refused("q_starts", call, host_rt, cache, replace(seqs, q_starts=buf(12)), total)
    refused("int32 offset", call, host_rt, cache, replace(seqs, num_seqs=1 << 31), total)
    for field in ("page_table", "kv_lens", "q_starts"):
        refused("4-byte aligned", call, host_rt, cache, replace(seqs, **{field: buf(4096, 2)}), total)


# ------------------------------------------------------------- attention ---

def test_attention_refuses(host_rt):
    cache, seqs, total = paged()
    for heads in (0, 3):
        refused("n_heads %d" % heads, call_attn, host_rt, cache, seqs, total, heads=heads)
    for s in (float("nan"), float("inf"), -3e38):
        refused("scale", call_attn, host_rt, cache, seqs, total, scale=s)
    refused("window needs causal", call_attn, host_rt, cache, seqs, total, causal=False, window=4)
    refused("attn_paged q", call_attn, host_rt, cache, seqs, total, q=buf(3 * 4 * 64 * 2 - 2))
    refused("attn_paged out", call_attn, host_rt, cache, seqs, total, out=buf(3 * 4 * 64 * 2 - 2))
    refused("aligned", call_attn, host_rt, cache, seqs, total, q=buf(1 << 20, 8))
    refused("aligned", call_attn, host_rt, cache, seqs, total, out=buf(1 << 20, 8))
    refused("aligned", call_attn, host_rt, cache, seqs, total, work=buf(1 << 27, 8))
    refused("256 values long but 255 apart", call_attn, host_rt, cache, seqs, total, q_stride=255)
    refused("not a multiple of 8", call_attn, host_rt, cache, seqs, total, q_stride=260)
    refused("workspace has 16 bytes", call_attn, host_rt, cache, seqs, total, work=buf(16))
    refused("overlap", call_attn, host_rt, cache, seqs, total, out=cache.k)
    refused("overlap", call_attn, host_rt, cache, seqs, total, work=nn.GpuBuffer(seqs.page_table.ptr & ~15, 1 << 27))
    one = buf(1 << 27)
    refused("overlap", call_attn, host_rt, cache, seqs, total, q=one, out=one)
    refused("overlap", call_attn, host_rt, cache, seqs, total, out=one, work=one)


def test_attention_refuses_more_than_it_counts(host_rt):
    """2^24 rows of 2^31 keys: more units of work than 32 bits count. The buffers are never touched."""
    big = 1 << 45
    cache = nn.PagedKv(nn.GpuBuffer(1 << 50, big), nn.GpuBuffer(1 << 51, big), 1 << 20, 2048, 1, 64)
    n = 1 << 24
    seqs = nn.PagedSeqs(nn.GpuBuffer(1 << 52, n * 8 << 20), nn.GpuBuffer(1 << 53, n * 4), None, n, 1 << 20)
    refused("more rows and keys", call_attn, host_rt, cache, seqs, n, heads=1, q=nn.GpuBuffer(1 << 54, big), out=nn.GpuBuffer(1 << 55, big))


def test_workspaces_grow_with_what_they_hold(host_rt):
    cache, seqs, _ = paged()
    few = nn.attn_paged_workspace_bytes(host_rt, 3, 4, cache, seqs)
    assert few > 0 and few == nn.attn_paged_workspace_bytes(host_rt, 3, 8, cache, seqs)
    many = nn.attn_paged_workspace_bytes(host_rt, 3, 4, cache, replace(seqs, num_seqs=1000))
    assert many > few
    assert nn.attn_paged_workspace_bytes(host_rt, 900, 4, cache, replace(seqs, q_starts=buf(16))) > few
    for bad in (replace(cache, head_dim=60), replace(cache, n_kv_heads=0), replace(cache, n_kv_heads=3)):
        assert nn.attn_paged_workspace_bytes(host_rt, 3, 4, bad, seqs) == 0


def test_attention_over_no_sequences_is_done_at_once(host_rt):
    cache, seqs, _ = paged()
    call_attn(host_rt, cache, replace(seqs, num_seqs=0), 0, q=buf(16), out=buf(16))


# ---------------------------------------------------------------- append ---

def test_append_refuses(host_rt):
    cache, seqs, total = paged()
    plan = nn.Rope(buf(32 * 8), 64, False, 1.0)
    norm = nn.QkNorm(buf(256), buf(256), 1e-6)
    refused("rot_dim 66", call_append, host_rt, cache, seqs, total, rope=replace(plan, rot_dim=66))
    refused("rope steps", call_append, host_rt, cache, seqs, total, rope=replace(plan, steps=buf(8)))
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        refused("eps", call_append, host_rt, cache, seqs, total, norm=replace(norm, eps=eps))
    refused("q norm weight", call_append, host_rt, cache, seqs, total, norm=replace(norm, q_weight=buf(252)))
    refused("k norm weight", call_append, host_rt, cache, seqs, total, norm=replace(norm, k_weight=buf(252)))
    refused("norm weights must be", call_append, host_rt, cache, seqs, total, norm=replace(norm, k_weight=buf(4096, 2)))
    for name in ("q", "k", "v", "q_out"):
        refused("kv_append_paged " + name, call_append, host_rt, cache, seqs, total, **{name: buf(64)})
        refused("not aligned", call_append, host_rt, cache, seqs, total, **{name: buf(1 << 20, 1)})
    refused("rows of k are 128 values long but 127", call_append, host_rt, cache, seqs, total, k_stride=127)
    refused("overlap", call_append, host_rt, cache, seqs, total, k=nn.GpuBuffer(cache.k.ptr, 1 << 20))
    refused("overlap", call_append, host_rt, replace(cache, v=cache.k), seqs, total)
    refused("overlap", call_append, host_rt, cache, seqs, total, q_out=nn.GpuBuffer(cache.v.ptr, 1 << 20))
    refused("too many heads", call_append, host_rt, cache, seqs, total, heads=(1 << 20) + 2)


def test_append_of_nothing_is_done_at_once(host_rt):
    cache, seqs, _ = paged()
    call_append(host_rt, cache, replace(seqs, num_seqs=0), 0)


# ---------------------------------------------------- native against ctypes ---

@pytest.mark.parametrize("name", capi.NATIVE_ATTENTION)
def test_native_and_ctypes_calls_refuse_alike(host_rt, name, monkeypatch):
    cache, seqs, total = paged()
    call = {"rope": lambda: call_rope(host_rt, **{**rope_args(), "x_stride": 100}),
            "kv_append_paged": lambda: call_append(host_rt, cache, seqs, total, k_stride=127),
            "attn_paged": lambda: call_attn(host_rt, cache, seqs, total, q_stride=260)}[name]
    with pytest.raises(nn.TesslError) as native:
        call()
    monkeypatch.setattr(nn._native, name, lambda *a: False)
    with pytest.raises(nn.TesslError) as plain:
        call()
    assert str(native.value) == str(plain.value)


def test_another_thread_is_refused(host_rt):
    import threading

    seen = []
    cache, seqs, total = paged()

    def go():
        try:
            call_attn(host_rt, cache, seqs, total)
        except nn.TesslError as e:
            seen.append(str(e))

    t = threading.Thread(target=go)
    t.start()
    t.join()
    assert "thread" in seen[0]
