"""The paged operators at the sizes where their kernels take another form:
rotations of many rows, appends and reads of several items a thread, the C
structs of a caller without the torch binding, and calls on two streams and in
two graphs for each form of attention.  Tolerances: test_kv4_gpu.py."""
import ctypes
import math

import numpy as np
import pytest
import torch

from test_kv4_gpu import HALF_STEP, TYPES, make, quantize_ref

pytestmark = pytest.mark.gpu


@pytest.fixture
def gen(rq_ctx):
    return torch.Generator(device="cuda").manual_seed(31)


def rotated(x, w, cos, sin, pos, rot, inter):
    """In 64 bits, from the formula."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    p = pos.clamp(0, cos.shape[0] - 1).long()
    c, s = cos.double()[p][:, None], sin.double()[p][:, None]
    i = torch.arange(0, rot, 2, device="cuda") if inter else torch.arange(rot // 2, device="cuda")
    j = i + (1 if inter else rot // 2)
    r = y.clone()
    r[..., i], r[..., j] = y[..., i] * c - y[..., j] * s, y[..., i] * s + y[..., j] * c
    return r


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("n,H,kv,hd,rot,weights", [
    (1301, 24, 8, 128, 128, "qk"), (2003, 19, 7, 96, 48, "q"), (1201, 12, 5, 256, 256, "k"), (5003, 31, 0, 32, 32, "qk"), (2503, 28, 4, 64, 16, ""),
])
def test_rotation_of_many_rows(gen, kind, inter, n, H, kv, hd, rot, weights):
    """More than 2^19 units of 8 elements: the form that takes two heads a
    group of lanes.  Odd head counts, padding, positions behind the tables, in
    place inside a packed matrix."""
    from rustyllm_b200.rope import qk_norm_rope, rope_tables
    assert n * (H + kv) * (hd // 8) > 606208
    flat = torch.randn(n, H + 2 * kv, hd, generator=gen, device="cuda").to(TYPES[kind])
    q, k = flat[:, :H], flat[:, H:H + kv]
    cos, sin = rope_tables(700, rot)
    pos = torch.randint(0, 700, (n,), generator=gen, device="cuda").to(torch.int32)
    pos[3], pos[n - 1], pos[n // 2] = -1, 700, 2 ** 31 - 1
    live = (pos >= 0) & (pos < 700)
    w = [1 + 0.1 * torch.randn(hd, generator=gen, device="cuda") if x in weights else None for x in "qk"]
    want = [rotated(x, y, cos, sin, pos, rot, inter) for x, y in zip((q, k), w)]
    keep = flat.clone()
    out = [torch.full_like(x.contiguous(), 3.0) for x in (q, k)]
    qk_norm_rope(q, k, pos, cos, sin, q_weight=w[0], k_weight=w[1], interleaved=inter, q_out=out[0], k_out=out[1])
    assert torch.equal(flat, keep)
    for got, x in zip(out, want):
        if x.numel():
            tol = (HALF_STEP[kind] + 8 * 2.0 ** -24) * x.abs() + 8 * 2.0 ** -24 * x.abs().amax(-1, keepdim=True).clamp(min=1e-6)
            assert ((got.double() - x).abs() <= tol)[live].all()
        assert (got[~live] == 3).all()
    qk_norm_rope(q, k, pos, cos, sin, q_weight=w[0], k_weight=w[1], interleaved=inter, q_out=q, k_out=k)
    assert torch.equal(q[live], out[0][live]) and torch.equal(k[live], out[1][live])
    assert torch.equal(flat[~live], keep[~live]) and torch.equal(flat[:, H + kv:], keep[:, H + kv:])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,hd,page,n", [(8, 128, 64, 5001), (12, 128, 16, 37), (3, 96, 32, 17003), (1, 32, 16, 152001), (20, 64, 16, 4001)])
def test_append_and_read_of_several_items_a_thread(gen, kind, kv, hd, page, n):
    from rustyllm_b200.kv4 import KV4Cache
    pages = (n + page - 1) // page + 1
    cache = KV4Cache(pages, page, kv, hd)
    k, v = make(gen, n, kv, hd, kind)
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n].to(torch.int32)
    given = slots.clone()
    given[n // 3], given[n - 1] = -1, pages * page  # not appended
    cache.append(k, v, given)
    for got, x in zip(cache.read(slots), (k, v)):
        want = quantize_ref(x.float().cpu().numpy())
        want[n // 3] = want[n - 1] = 0
        assert np.array_equal(got.cpu().numpy().astype(np.float64), want)
    every = torch.arange(pages * page, dtype=torch.int32, device="cuda")
    whole = cache.read(every)
    for t in ("f16", "bf16"):
        for a, b in zip(cache.read(every, TYPES[t]), whole):
            assert torch.equal(a, b.to(TYPES[t]))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,kv,hd,rot,inter", [(32, 8, 128, 128, False), (5, 1, 96, 32, True), (3, 3, 32, 32, False)])
def test_rotation_with_append_of_many_tokens(gen, kind, H, kv, hd, rot, inter):
    """Queries and values as the formula and the cache's rule give them, keys
    within the bound of test_kv4_gpu's comparison of one pass and two; q, k
    and v side by side, q written in place, padding left alone."""
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.rope import qk_norm_rope, qk_norm_rope_append, rope_tables
    n = 701
    flat = torch.randn(n, H + 2 * kv, hd, generator=gen, device="cuda").to(TYPES[kind])
    q, k, v = flat[:, :H], flat[:, H:H + kv], flat[:, H + kv:]
    keep = flat.clone()
    cos, sin = rope_tables(900, rot)
    pos = torch.randint(0, 900, (n,), generator=gen, device="cuda").to(torch.int32)
    pos[5], pos[n - 1] = -1, 900
    live = (pos >= 0) & (pos < 900)
    slots = torch.randperm(800, generator=gen, device="cuda")[:n].to(torch.int32)
    w = [1 + 0.1 * torch.randn(hd, generator=gen, device="cuda") for _ in range(2)]
    want = rotated(q, w[0], cos, sin, pos, rot, inter)
    two = KV4Cache(50, 16, kv, hd)
    two.append(qk_norm_rope(q, k, pos, cos, sin, q_weight=w[0], k_weight=w[1], interleaved=inter)[1], v,
               torch.where(live, slots, -1))
    one = KV4Cache(50, 16, kv, hd)
    qk_norm_rope_append(one, q, k, v, pos, slots, cos, sin, q_weight=w[0], k_weight=w[1], interleaved=inter, q_out=q)
    tol = (HALF_STEP[kind] + 8 * 2.0 ** -24) * want.abs() + 8 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True)
    assert ((q.double() - want).abs() <= tol)[live].all()
    assert torch.equal(flat[~live], keep[~live]) and torch.equal(flat[:, H:], keep[:, H:])
    every = torch.arange(800, dtype=torch.int32, device="cuda")
    (a, b), (c, d) = one.read(every), two.read(every)
    assert torch.equal(b, d)
    step = c.unflatten(2, (-1, 32)).abs().amax(-1, keepdim=True) / 8
    off = (a - c).unflatten(2, (-1, 32)).abs()
    assert (off <= step * (1 + 9 * (HALF_STEP[kind] + 2.0 ** -10))).all()


@pytest.mark.parametrize("kind,nq,group", [("f32", 3, 8), ("f32", 20, 8), ("f16", 1, 8), ("bf16", 2, 8), ("bf16", 9, 4), ("bf16", 40, 8)])
def test_each_form_on_two_streams_and_in_two_graphs(gen, kind, nq, group):
    """The same bits alone, beside another call and replayed: no call's pieces
    or operands meet another's.  (The last two are the forms on tcgen05.)"""
    from rustyllm_b200.kv4 import KV4Cache
    B, n = 3, 1500
    cache = KV4Cache(B * 94, 16, 2, 64)
    k, v = make(gen, B * 94 * 16, 2, 64, kind)
    cache.append(k, v, torch.arange(B * 94 * 16, dtype=torch.int32, device="cuda"))
    table = torch.randperm(B * 94, generator=gen, device="cuda").to(torch.int32).view(B, 94)
    lens = torch.tensor([n, 77, 1200], dtype=torch.int32, device="cuda")
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda") * nq
    qs = [torch.randn(B * nq, 2 * group, 64, generator=gen, device="cuda").to(TYPES[kind]) for _ in range(2)]

    def call(q):
        return cache.attention(q, table, lens, cu_q=cu, max_q=nq)

    want = [call(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(10):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(call(q))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for q, s in zip(qs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(call(q))
        graphs.append(g)
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    del graphs


def test_the_c_structs_alone(gen):
    """A caller that fills rq_kv4_query and rq_qk_rope itself."""
    from rustyllm_b200 import Context, _lib
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.rope import qk_norm_rope, rope_tables
    lib, ctx = _lib.lib(), Context.get(0)
    n, H, kv, hd = 6, 4, 2, 64
    cache = KV4Cache(4, 16, kv, hd)
    k, v = make(gen, 64, kv, hd, "f16")
    cache.append(k, v, torch.arange(64, dtype=torch.int32, device="cuda"))
    q = torch.randn(n, H, hd, generator=gen, device="cuda").half()
    cos, sin = rope_tables(100, hd)
    pos = torch.arange(50, 50 + n, dtype=torch.int32, device="cuda")
    want_q, want_k = qk_norm_rope(q, k[:n], pos, cos, sin)
    qo, ko = torch.zeros_like(q), torch.zeros_like(k[:n])
    torch.cuda.synchronize()
    pair = ctypes.c_int64 * 2
    a = _lib.QkRope(dtype=_lib.RQ_F16, n_tokens=n, n_heads=H, n_kv_heads=kv, head_dim=hd, rot_dim=hd, q=q.data_ptr(), q_stride=pair(H * hd, hd),
                    q_out=qo.data_ptr(), q_out_stride=pair(H * hd, hd), k=k.data_ptr(), k_stride=pair(kv * hd, hd), k_out=ko.data_ptr(),
                    k_out_stride=pair(kv * hd, hd), eps=1e-6, cos=cos.data_ptr(), sin=sin.data_ptr(), max_pos=100, positions=pos.data_ptr())
    _lib.check(lib.rq_qk_norm_rope(ctx.handle, ctypes.byref(a), None))
    torch.cuda.synchronize()
    assert torch.equal(qo, want_q) and torch.equal(ko, want_k)
    for name, value, msg in (("head_dim", 63, "head_dim 63"), ("rot_dim", 66, "rot_dim 66"), ("dtype", 7, "dtype 7"), ("q", None, "q is NULL"),
                             ("n_heads", -1, "heads"), ("max_pos", 0, "max_pos"), ("k_out_stride", pair(hd, hd), "lie on one another")):
        keep = getattr(a, name)
        keep = pair(*keep) if name.endswith("stride") else keep
        setattr(a, name, value)
        assert lib.rq_qk_norm_rope(ctx.handle, ctypes.byref(a), None) != 0 and msg in _lib.last_error(), name
        setattr(a, name, keep)
    table = torch.arange(4, dtype=torch.int32, device="cuda")
    lens = torch.tensor([60], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    want = cache.attention(q, table[None], lens, cu_q=cu, max_q=n)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    b = _lib.Kv4Query(dtype=_lib.RQ_F16, q=q.data_ptr(), q_stride=pair(H * hd, hd), out=out.data_ptr(), out_stride=pair(H * hd, hd), n_tokens=n,
                      n_heads=H, batch=1, max_q=n, cu_q=cu.data_ptr(), kv_lens=lens.data_ptr(), block_table=table.data_ptr(), table_stride=4,
                      table_width=4, scale=hd ** -0.5)
    need = ctypes.c_size_t()
    _lib.check(lib.rq_kv4_attention_workspace(cache.handle, ctypes.byref(b), ctypes.byref(need)))
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    b.workspace, b.workspace_bytes = ws.data_ptr(), need.value
    _lib.check(lib.rq_kv4_attention(cache.handle, ctypes.byref(b), None))
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    if need.value:
        for pointer, size in ((None, need.value), (ws.data_ptr() + 4, need.value), (ws.data_ptr(), need.value - 1)):
            b.workspace, b.workspace_bytes = pointer, size
            assert lib.rq_kv4_attention(cache.handle, ctypes.byref(b), None) != 0 and "workspace" in _lib.last_error()
        b.workspace, b.workspace_bytes = ws.data_ptr(), need.value
    for name, value, msg in (("n_heads", 3, "3 query heads"), ("max_q", 0, "max_q 0"), ("scale", math.inf, "scale"), ("kv_lens", None, "kv_lens is NULL"),
                             ("out_stride", pair(hd, hd), "lie on one another"), ("table_width", 2 ** 28, "2^31")):
        keep = getattr(b, name)
        keep = pair(*keep) if name.endswith("stride") else keep
        setattr(b, name, value)
        assert lib.rq_kv4_attention(cache.handle, ctypes.byref(b), None) != 0 and msg in _lib.last_error(), name
        setattr(b, name, keep)
