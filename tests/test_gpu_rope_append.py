"""rope and kv_append_paged against their definitions in 64 bits: layouts, types, far positions, strides, in place, the cache's other
slots left as they were, tokens without a place, ids outside; and the run that they belong to, from a fused projection to the
attention's output."""
import numpy as np
import pytest

from gpu_util import rt, upload_bank  # noqa: F401
from paged_util import NAN16, SENTINEL16, U16, U32, Batch, bf16, f64, normed, turn, turn_size
from tessl_b200 import nn, synth

pytestmark = pytest.mark.gpu
THETA = 1e7


def stored(want, size, as16, extra=0.0):
    """Tolerance of a turned value: two products and a sum in f32 of cosines and sines that are off by 4 U32 (fraction of a turn to
    f32, function), `extra` relative error of the inputs; then the rounding of the result."""
    off = size * (8 * U32 + extra)
    return off + ((U16 if as16 else U32) * (np.abs(want) + off)) + 1e-38


def as_input(a, as16):
    return (bf16(a), f64(bf16(a))) if as16 else (np.asarray(a, np.float32), np.asarray(a, np.float32).astype(np.float64))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("x16,out16", [(False, False), (False, True), (True, True), (True, False)])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 40, 128, 128), (33, 3, 64, 32), (700, 1, 96, 24), (5, 7, 256, 64), (9, 2, 20, 20),
                                                  (4, 5, 2, 2), (6, 3, 250, 130), (3, 2, 128, 0), (2, 600, 8, 8)])
def test_rope(rt, tokens, heads, dim, rot, x16, out16, interleaved):
    r = np.random.default_rng(tokens * 1000 + dim)
    x, xf = as_input(r.standard_normal((tokens, heads, dim)), x16)
    pos = r.integers(-2**31, 2**31, tokens).astype(np.int32)
    pos[: tokens // 2] = r.integers(0, 200000, tokens // 2)
    plan = nn.rope_plan(rt, rot, THETA, interleaved=interleaved)
    out = rt.buffer_from(np.full(x.size + 32, SENTINEL16, np.uint16 if out16 else np.uint32))
    size = 2 if out16 else 4
    nn.rope(rt, rt.buffer_from(x), rt.buffer_from(pos), out.view(0, x.size * size), plan, tokens, heads, dim, x16, out16)
    got = out.read(np.uint16 if out16 else np.uint32, x.size + 32)
    assert (got[x.size:] == SENTINEL16).all()
    g = (f64(got[:x.size]) if out16 else got[:x.size].view(np.float32).astype(np.float64)).reshape(x.shape)
    # the steps are whole multiples of 2^-64 turns: at position 2^31 that is 2^-34 turns, less than U32
    want = turn(xf, pos, rot, THETA, interleaved)
    # angles of 64 bits at 2^31 radians are themselves off by 2^-22
    slack = np.abs(pos.astype(np.float64))[:, None, None] * 2.0 ** -52
    assert (np.abs(g - want) <= stored(want, turn_size(xf, rot, interleaved), out16, 2 * slack)).all()


@pytest.mark.parametrize("x16", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_in_place_and_in_wider_rows(rt, x16, interleaved):
    tokens, heads, dim, rot, stride = 50, 6, 64, 32, 6 * 64 + 12
    r = np.random.default_rng(3)
    x, xf = as_input(r.standard_normal((tokens, stride)), x16)
    pos = np.arange(1000, 1000 + tokens).astype(np.int32)
    plan = nn.rope_plan(rt, rot, THETA, interleaved=interleaved)
    b = rt.buffer_from(x)
    nn.rope(rt, b, rt.buffer_from(pos), b, plan, tokens, heads, dim, x16, x16, stride, stride)
    got = b.read(x.dtype, x.size).reshape(x.shape)
    assert np.array_equal(got[:, heads * dim:], x[:, heads * dim:]), "between the rows nothing is written"
    v = xf[:, :heads * dim].reshape(tokens, heads, dim)
    g = got[:, :heads * dim]
    g = (f64(g) if x16 else g.astype(np.float64)).reshape(v.shape)
    want = turn(v, pos, rot, THETA, interleaved)
    assert (np.abs(g - want) <= stored(want, turn_size(v, rot, interleaved), x16)).all()
    # rows that start anywhere: the same bits
    for shift in (1, 2):
        size = x.itemsize
        flat = np.zeros(x.size + 8, x.dtype)
        flat[shift:shift + x.size] = x.reshape(-1)
        b = rt.buffer_from(flat)
        at = b.view(shift * size, x.size * size)
        nn.rope(rt, at, rt.buffer_from(pos), at, plan, tokens, heads, dim, x16, x16, stride, stride)
        assert np.array_equal(b.read(x.dtype, flat.size)[shift:shift + x.size].reshape(x.shape), got)


@pytest.mark.parametrize("kind", ["linear", "ntk", "wavelength", "yarn"])
def test_rope_scaled(rt, kind):
    tokens, heads, dim = 20, 2, 128
    x = np.random.default_rng(4).standard_normal((tokens, heads, dim)).astype(np.float32)
    pos = (np.arange(tokens) * 9973).astype(np.int32)
    scaling = nn.RopeScaling(kind, 8.0, 8192.0)
    plan = nn.rope_plan(rt, dim, 500000.0, scaling=scaling)
    steps, factor = nn.rope_steps(dim, 500000.0, scaling)
    out = rt.alloc_buffer(x.nbytes)
    nn.rope(rt, rt.buffer_from(x), rt.buffer_from(pos), out, plan, tokens, heads, dim, False, False)
    w = steps.astype(np.float64) * 2.0 ** -64 * 2 * np.pi
    xf = x.astype(np.float64)
    want = turn(xf, pos, dim, None, False, factor, w)
    g = out.read(np.float32, x.size).reshape(x.shape).astype(np.float64)
    assert (np.abs(g - want) <= stored(want, turn_size(xf, dim, False, factor), False)).all()


# lens, news, kv heads, group, dim, page, head major, rot, norm, in16
APPENDS = [
    ([5], [1], 1, 1, 64, 16, False, 64, False, False),
    ([100, 64, 65, 1], [1, 1, 1, 1], 4, 4, 256, 64, False, 64, True, False),
    ([100, 30, 0, 17], [60, 30, 0, 3], 8, 4, 128, 16, True, 128, False, True),
    ([300, 20], [300, 19], 2, 3, 96, 7, False, 24, True, True),
    ([40, 33], [1, 33], 1, 1, 8, 1, True, 8, True, False),
    ([40, 33], [40, 3], 3, 2, 72, 48, False, 36, True, False),   # runs that are no multiple of four pairs
    ([40, 33], [4, 3], 3, 2, 200, 48, True, 0, False, True),
    ([2, 9], [5, 9], 2, 2, 128, 4, False, 128, True, False),      # tokens before position 0
]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(rt, case, fused):
    lens, news, kvh, g, d, page, hm, rot, norm, in16 = APPENDS[case]
    b = Batch(200 + case, lens, news, kvh, g, d, page, hm, tail=2)
    run_append(rt, b, rot, norm, in16, fused, 0, case % 2 == 1)


def run_append(rt, b, rot, norm, in16, fused, pad, interleaved, holes=()):
    r, h, kvh, d, n = b.rng, b.heads, b.kv_heads, b.dim, b.total
    x, xf = as_input(r.standard_normal((n, (h + 2 * kvh) * d + pad)) * 1.7, in16)
    size = x.itemsize
    b.upload(rt)
    k0, v0 = b.k.copy(), b.v.copy()
    wq, wk = (r.standard_normal(d).astype(np.float32) * np.float32(0.1) for _ in range(2))
    plan = nn.rope_plan(rt, rot, THETA, interleaved=interleaved) if rot else None
    norms = nn.QkNorm(rt.buffer_from(wq), rt.buffer_from(wk), 1e-6) if norm else None
    if fused:
        buf, s = rt.buffer_from(x), x.shape[1]
        nq, nk = h * d, kvh * d
        q, k, v = (buf.view(o * size, ((n - 1) * s + w) * size) for o, w in ((0, nq), (nq, nk), (nq + nk, nk)))
        strides = (s, s, s)
    else:
        parts = x[:, :h * d], x[:, h * d:(h + kvh) * d], x[:, (h + kvh) * d:(h + 2 * kvh) * d]
        q, k, v = (rt.buffer_from(np.ascontiguousarray(p)) for p in parts)
        strides = (0, 0, 0)
    nn.kv_append_paged(rt, q, k, v, b.out.view(0, b.q.size * 2), b.cache, b.seqs, plan, norms, n, h, *strides, in16)
    got_q = b.out.read(np.uint16, b.q.size + 64)
    live = b.live * h * d
    assert (got_q[live:] == SENTINEL16).all(), "rows that belong to no sequence were written"
    xf = xf[:, :(h + 2 * kvh) * d].reshape(n, h + 2 * kvh, d)[:b.live]
    qf, kf, vf = xf[:, :h], xf[:, h:h + kvh], xf[:, h + kvh:]
    pos = np.concatenate([np.arange(l - m, l) for l, m in zip(b.lens, b.news)]).astype(np.int64)
    extra = 0.0
    if norm:  # the mean of d squares, root, division, two products
        qf, kf, extra = normed(qf, wq.astype(np.float64), 1e-6), normed(kf, wk.astype(np.float64), 1e-6), (d + 8) * U32
    for name, got, src in (("q", f64(got_q[:live]).reshape(qf.shape), qf),):
        want = turn(src, pos, rot, THETA, interleaved)
        assert (np.abs(got - want) <= stored(want, turn_size(src, rot, interleaved), True, extra)).all(), name
    got_k, got_v = b.b_k.read(np.uint16, b.k.size).reshape(b.k.shape), b.b_v.read(np.uint16, b.v.size).reshape(b.v.shape)
    want_k = turn(kf, pos, rot, THETA, interleaved)
    tol_k = stored(want_k, turn_size(kf, rot, interleaved), True, extra)
    want_v = bf16(vf)
    written = np.zeros(b.k.shape, bool)
    row = 0
    for s in range(b.n):
        for i in range(b.news[s]):
            p = b.lens[s] - b.news[s] + i
            if p >= 0 and (s, p // b.page) not in holes and p < b.width * b.page:
                page, slot = b.table[s, p // b.page], p % b.page
                at = (page, slice(None), slot) if b.head_major else (page, slot)
                assert (np.abs(f64(got_k[at]) - want_k[row]) <= tol_k[row]).all(), ("k", s, i)
                assert np.array_equal(got_v[at], want_v[row]), ("v", s, i)
                written[at] = True
            row += 1
    assert np.array_equal(got_k[~written], k0[~written]) and np.array_equal(got_v[~written], v0[~written]), "other slots were written"


def test_append_leaves_out_what_has_no_place(rt):
    """Ids outside the cache, and positions past the table's row: their queries are made, nothing is stored."""
    b = Batch(21, [40, 20], [30, 20], 2, 2, 64, 8)
    b.table[0, 2], b.table[1, 1] = b.pages, -1
    run_append(rt, b, 64, False, False, True, 4, False, holes=[(0, 2), (1, 1)])
    b = Batch(22, [40, 20], [30, 20], 2, 2, 64, 8)
    b.table, b.width = np.ascontiguousarray(b.table[:, :4]), 4
    run_append(rt, b, 64, True, True, False, 0, False)


def test_append_without_queries(rt):
    b = Batch(23, [9, 30], [4, 30], 2, 2, 64, 16).upload(rt)
    x = [np.random.default_rng(i).standard_normal((b.total, 2 * 64)).astype(np.float32) for i in range(2)]
    nn.kv_append_paged(rt, None, rt.buffer_from(x[0]), rt.buffer_from(x[1]), None, b.cache, b.seqs, None, None, b.total, 0)
    got = b.b_v.read(np.uint16, b.v.size).reshape(b.v.shape)
    b.put("v", 0, 5, bf16(x[1][:4]).reshape(4, 2, 64)), b.put("v", 1, 0, bf16(x[1][4:]).reshape(30, 2, 64))
    assert np.array_equal(got, b.v)
    assert np.array_equal(b.b_k.read(np.uint16, b.k.size).reshape(b.k.shape)[b.table[1, 0], :], bf16(x[0][4:20]).reshape(16, 2, 64))


def test_many_sequences_find_their_rows(rt):
    news = [(i * 7) % 3 for i in range(1500)]
    lens = [n + (i * 13) % 9 for i, n in enumerate(news)]
    b = Batch(24, lens, news, 1, 1, 16, 4, tail=1)
    run_append(rt, b, 16, False, False, True, 0, False)


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 1, 9]])
@pytest.mark.parametrize("graph", [False, True])
def test_projection_to_attention(rt, news, graph):
    """q/k/v projection, append, attention, output projection, one behind the other on the runtime's stream: every operator gives the
    bits that it gives when each call is waited for; and the attention's output is that of its definition over the cache it read."""
    import torch

    hidden, kvh, g, d, page = 1024, 2, 4, 128, 16
    lens, total = [300, 70, 41], sum(news)
    b = Batch(25, lens, news, kvh, g, d, page).upload(rt)
    rows = (b.heads + 2 * kvh) * d
    qkv_bank, o_bank = upload_bank(rt, *synth.q4_bank(0x7E551600, rows, hidden, 64)), upload_bank(rt, *synth.q4_bank(0x7E551601, hidden, b.heads * d, 64))
    x = rt.buffer_from(synth.normal_bf16(0x7E551602, total * hidden))
    qkv, q16 = rt.alloc_buffer(total * rows * 4), rt.alloc_buffer(b.q.size * 2)
    out, y = rt.alloc_buffer(b.q.size * 2), rt.alloc_buffer(total * hidden * 4)
    plan = nn.rope_plan(rt, 64, THETA)
    norms = nn.QkNorm(rt.buffer_from(np.zeros(d, np.float32)), rt.buffer_from(np.zeros(d, np.float32)), 1e-6)
    work = rt.alloc_buffer(nn.attn_paged_workspace_bytes(rt, total, b.heads, b.cache, b.seqs))
    qw, kw = b.heads * d * 4, kvh * d * 4
    rest = (total - 1) * rows * 4
    views = [qkv.view(0, rest + qw), qkv.view(qw, rest + kw), qkv.view(qw + kw, rest + kw)]

    def project(bank, a, c, shape):
        if total <= nn.GEMM_Q4_MLX_MAX_M:
            nn.gemm_q4_mlx(rt, bank, a, c, shape, total)
        else:
            nn.gemm_q4_mlx_tensorops(rt, bank, a, c, shape, total)

    def chain():
        project(qkv_bank, x, qkv, nn.QuantShape(rows, hidden, 64))
        nn.kv_append_paged(rt, *views, q16, b.cache, b.seqs, plan, norms, total, b.heads, rows, rows, rows)
        nn.attn_paged(rt, q16, b.cache, b.seqs, out, work, total, b.heads, d ** -0.5)
        project(o_bank, out, y, nn.QuantShape(hidden, b.heads * d, 64))

    chain()
    rt.synchronize()
    want = {n: t.read(np.uint16, t.nbytes // 2) for n, t in (("q", q16), ("out", out), ("y", y), ("k", b.b_k), ("v", b.b_v))}
    b.q, b.k, b.v = want["q"].reshape(b.q.shape), want["k"].reshape(b.k.shape), want["v"].reshape(b.v.shape)
    b.check(np.concatenate([want["out"], np.full(64, SENTINEL16, np.uint16)]))
    rt.set_encode_only(True)
    try:
        for t in (q16, out, y, qkv):
            t.write(np.zeros(t.nbytes, np.uint8))
        if graph:
            cg = torch.cuda.CUDAGraph()
            with torch.cuda.graph(cg, stream=torch.cuda.ExternalStream(rt.stream)):
                chain()
            with torch.cuda.stream(torch.cuda.ExternalStream(rt.stream)):
                for _ in range(3):
                    cg.replay()
        else:
            for _ in range(3):
                chain()
        rt.synchronize()
        for n, t in (("q", q16), ("out", out), ("y", y), ("k", b.b_k), ("v", b.b_v)):
            assert np.array_equal(t.read(np.uint16, t.nbytes // 2), want[n]), n
    finally:
        rt.set_encode_only(False)
