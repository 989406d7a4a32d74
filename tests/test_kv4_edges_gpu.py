"""The paged operators where values, sizes and arguments are extreme, against
the plain implementations (and the tolerances) of test_kv4_gpu.py."""
import math

import numpy as np
import pytest
import torch

from test_kv4_gpu import TYPES, attention_ref, close, make, quantize_ref

pytestmark = pytest.mark.gpu


@pytest.fixture
def gen(rq_ctx):
    return torch.Generator(device="cuda").manual_seed(23)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Setup:
    """One sequence of n positions in pages of 16 that lie in random order,
    and its last nq queries."""

    def __init__(self, gen, kind, n, nq, kv, group, hd, k, v, q=None, scale=None, window=0):
        from rustyllm_b200.kv4 import KV4Cache
        self.n, self.nq, self.window, self.scale = n, nq, window, hd ** -0.5 if scale is None else scale
        width = (n + 15) // 16
        self.cache = KV4Cache(width + 1, 16, kv, hd)
        self.table = torch.randperm(width + 1, generator=gen, device="cuda")[:width].to(torch.int32)[None].contiguous()
        j = torch.arange(n, device="cuda")
        self.slots = (self.table[0, j // 16] * 16 + j % 16).to(torch.int32)
        self.cache.append(k, v, self.slots)
        self.q = torch.randn(nq, kv * group, hd, generator=gen, device="cuda").to(TYPES[kind]) if q is None else q

    def call(self):
        return self.cache.attention(self.q, self.table, i32(self.n), cu_q=i32(0, self.nq), max_q=self.nq, scale=self.scale,
                                    window=self.window)

    def want(self):
        every = torch.arange(self.cache.n_pages * 16, dtype=torch.int32, device="cuda")
        rk, rv = (x.double().cpu().numpy() for x in self.cache.read(every))
        return attention_ref(self.q.double().cpu().numpy(), rk, rv, self.table.cpu().numpy(), 16, [self.n], [0, self.nq],
                             self.scale, self.window, self.cache.n_pages)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 3, 21])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_value_without_weight_costs_no_bits(gen, kind, nq, hd):
    """The largest value that the cache can hold, at a position that every
    query sees and none weighs (its score lies over 60 below the others'),
    beside values of 0.05.  4 rows a kv head, 12 and 84: each form."""
    n = 500
    k, v = make(gen, n, 2, hd, kind)
    v = (v.float() * 0.1).to(TYPES[kind])
    q = torch.randn(nq, 8, hd, generator=gen, device="cuda").abs().to(TYPES[kind])
    k[3] = -20
    v[3] = 6e4 if kind == "f16" else 5.2e5
    s = Setup(gen, kind, n, nq, 2, 4, hd, k, v, q)
    close(s.call(), s.want(), slice(None), kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 21])
@pytest.mark.parametrize("what", ["huge", "nan"])
def test_values_before_the_window_do_not_enter(gen, kind, nq, what):
    """The window of the first query starts inside a tile, behind a position
    of huge or not-a-number keys and values."""
    n, window = 300, 100
    first = n - nq - window + 1  # the first position that any query sees
    assert first % 16
    k, v = make(gen, n, 2, 64, kind)
    v = (v.float() * 0.1).to(TYPES[kind])
    s = Setup(gen, kind, n, nq, 2, 4, 64, k, v, window=window)
    want = s.want()
    k[first - 1] = v[first - 1] = math.nan if what == "nan" else 6e4 if kind == "f16" else 5.2e5
    s.cache.append(k, v, s.slots)
    close(s.call(), want, slice(None), kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [2, 21])
@pytest.mark.parametrize("what", ["huge", "nan"])
def test_values_that_the_last_query_alone_sees_do_not_enter_others(gen, kind, nq, what):
    n = 300
    k, v = make(gen, n, 2, 64, kind)
    v = (v.float() * 0.1).to(TYPES[kind])
    s = Setup(gen, kind, n, nq, 2, 4, 64, k, v)
    want = s.want()
    k[-1] = v[-1] = math.nan if what == "nan" else 6e4 if kind == "f16" else 5.2e5
    s.cache.append(k, v, s.slots)
    close(s.call()[:-1], want, slice(0, nq - 1), kind)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("nq", [1, 21])
@pytest.mark.parametrize("falls", [False, True])
def test_values_that_grow_or_fall_over_the_sequence(gen, kind, nq, falls):
    n = 400
    k, v = make(gen, n, 2, 96, kind)
    size = torch.logspace(-3.5, 3.5, n, device="cuda")
    v = (v.float() * (size.flip(0) if falls else size)[:, None, None]).to(TYPES[kind])
    s = Setup(gen, kind, n, nq, 2, 4, 96, k, v)
    close(s.call(), s.want(), slice(None), kind)


@pytest.mark.parametrize("nq", [1, 21])
@pytest.mark.parametrize("size", [2.0 ** -19, 2.0 ** -16, 2.0 ** 14])
def test_f32_accuracy_at_the_ends_of_the_scales(gen, nq, size):
    """Scales down among f16's smallest numbers and up to its largest."""
    k, v = make(gen, 200, 2, 64, "f32")
    s = Setup(gen, "f32", 200, nq, 2, 4, 64, k, v * size)
    got, want = s.call().double().cpu().numpy(), s.want()[0]
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < 2e-6


def test_values_of_zero_next_to_others(gen):
    """Positions without value still count in the sum of weights, however far
    above the others their scores lie."""
    k, v = make(gen, 100, 2, 64, "f32")
    v[10:60] = 0
    k[20] = 6
    q = torch.randn(2, 8, 64, generator=gen, device="cuda").abs()
    s = Setup(gen, "f32", 100, 2, 2, 4, 64, k, v, q)
    close(s.call(), s.want(), slice(None), "f32")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_finite_values_of_every_size_saturate_at_their_own_end(gen, kind):
    """Elements from 5e5, where a block's scale reaches its end, to the largest
    finite ones, of both signs, beside a larger one and a small one."""
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.rope import qk_norm_rope_append, rope_tables
    sizes = torch.logspace(math.log10(5e5), 38.4, 600, dtype=torch.float64).float().to(TYPES[kind])
    n = sizes.numel()
    k = torch.randn(n, 2, 64, generator=gen, device="cuda").to(TYPES[kind])
    sizes = sizes.cuda()
    for head, sign in ((0, 1), (1, -1)):
        k[:, head, 0], k[:, head, 33] = sign * sizes, sign * sizes
        k[:, head, 7], k[:, head, 40] = -sign * sizes, sign * sizes * 0.75
        k[1:, head, 9] = sign * sizes[:-1]
    v = k.flip(0).contiguous()
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    every = KV4Cache(n // 16 + 1, 16, 2, 64), KV4Cache(n // 16 + 1, 16, 2, 64)
    every[0].append(k, v, slots)
    q = torch.zeros(n, 2, 64, device="cuda", dtype=TYPES[kind])
    qk_norm_rope_append(every[1], q, k, v, slots % 4, slots, *rope_tables(4, 0))  # nothing is rotated
    for cache in every:
        for got, x in zip(cache.read(slots), (k, v)):
            assert np.array_equal(got.cpu().numpy().astype(np.float64), quantize_ref(x.double().cpu().numpy()))


@pytest.mark.parametrize("kind,kv,group", [("f32", 2, 1), ("bf16", 2, 1), ("f32", 1, 16), ("bf16", 1, 16), ("bf16", 1, 40)])
def test_sequences_of_more_queries_than_announced(gen, kind, kv, group):
    """The first max_q rows of each sequence at their own positions (two of
    them before the first one held), the others left as they were; without
    max_q all of them."""
    from rustyllm_b200.kv4 import KV4Cache
    n, lens = 4 + 18 + 7, [60, 100, 5]
    cache = KV4Cache(24, 16, kv, 64)
    k, v = make(gen, 24 * 16, kv, 64, kind)
    every = torch.arange(24 * 16, dtype=torch.int32, device="cuda")
    cache.append(k, v, every)
    rk, rv = (x.double().cpu().numpy() for x in cache.read(every))
    table = torch.randperm(24, generator=gen, device="cuda")[:21].view(3, 7).to(torch.int32)
    q = torch.randn(n, kv * group, 64, generator=gen, device="cuda").to(TYPES[kind])
    cu = [0, 4, 22, 29]
    want = attention_ref(q.double().cpu().numpy(), rk, rv, table.cpu().numpy(), 16, lens, cu, 0.125, 0, 24)
    for most in (4, 1):
        out = torch.full_like(q, 9.0)
        cache.attention(q, table, i32(*lens), cu_q=i32(*cu), max_q=most, out=out)
        first = [r for b in range(3) for r in range(cu[b], min(cu[b] + most, cu[b + 1]))]
        close(out[first], want, first, kind)
        rest = [r for r in range(n) if r not in first]
        assert (out[rest] == 9).all()
    close(cache.attention(q, table, i32(*lens), cu_q=i32(*cu)), want, slice(None), kind)
    # offsets that say anything at all: nothing outside the rows is read or written
    out = torch.full_like(q, 9.0)
    cache.attention(q, table, i32(*lens), cu_q=i32(-2 ** 31, 2 ** 31 - 1, 28, 29), max_q=4, out=out, window=2 ** 31 - 1)
    assert (out[:28] == 9).all() and out[28].isfinite().all()
    if kind == "f32":
        last = attention_ref(q.double().cpu().numpy(), rk, rv, table.cpu().numpy()[2:], 16, lens[2:], [28, 29], 0.125, 0, 24)
        close(out[28:], last, [28], kind)


def test_rows_past_32_bits_are_refused(gen):
    """2^38 rows of a kv head and some: their number of row tiles, cut to 32
    bits, would be a small one."""
    from rustyllm_b200 import RqError
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(1, 16, 1, 32)
    q = torch.zeros(1, 65536, 32, device="cuda")
    for most in (2 ** 22 + 16, 2 ** 24, 2 ** 15):
        with pytest.raises(RqError, match="too many rows"):
            cache.attention(q, i32(0)[None], i32(1), cu_q=i32(0, 1), max_q=most)
    assert not cache.attention(q, i32(0)[None], i32(1), cu_q=i32(0, 1), max_q=2).any()


def test_outputs_whose_rows_overlap_in_part_are_refused(gen):
    """Every layout of [tokens, heads] in which two rows share an element, and
    none of the others: transposed, inside a packed matrix, interleaved."""
    from rustyllm_b200 import RqError
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.rope import qk_norm_rope, qk_norm_rope_append, rope_tables
    cache = KV4Cache(2, 16, 2, 32)
    k, v = make(gen, 32, 2, 32, "f32")
    cache.append(k, v, torch.arange(32, dtype=torch.int32, device="cuda"))
    tables = rope_tables(8, 32)
    refused = 0
    for n, h in ((3, 4), (5, 2), (1, 4)):
        q = torch.randn(n, h, 32, generator=gen, device="cuda")
        pos = torch.arange(n, dtype=torch.int32, device="cuda")
        args = dict(cu_q=i32(0, n), max_q=n)
        table, lens = i32(0, 1)[None], i32(20)
        plain = cache.attention(q, table, lens, **args), *qk_norm_rope(q, k[:n], pos, *tables)
        for st, sh in ((32, 32 * n), (32 * h, 32), (31, 200), (200, 31), (64, 32), (96, 64), (64, 96), (64, 95), (96, 33), (160, 64), (80, 48),
                       (32 * h - 1, 32), (7 * 32, 40), (0, 32)):
            cells = torch.zeros(n, h, 32, dtype=torch.int64)
            at = (torch.arange(n)[:, None, None] * st + torch.arange(h)[:, None] * sh + torch.arange(32) + cells).reshape(-1)
            apart = at.unique().numel() == at.numel()
            out = torch.zeros(4096, device="cuda").as_strided((n, h, 32), (st, sh, 1))
            calls = (lambda: cache.attention(q, table, lens, out=out, **args),
                     lambda: qk_norm_rope(q, k[:n], pos, *tables, q_out=out)[0],
                     lambda: qk_norm_rope_append(cache, q, k[:n], v[:n], pos, pos - 40, *tables, q_out=out),
                     lambda: qk_norm_rope(k[:n], q, pos, *tables, k_out=out)[1])
            for call, want in zip(calls, (plain[0], plain[1], plain[1], plain[1])):
                if apart:
                    assert torch.allclose(call(), want, rtol=1e-5, atol=1e-5)
                else:
                    refused += 1
                    with pytest.raises(RqError, match="lie on one another"):
                        call()
    assert refused == 60  # 15 of the 42 layouts


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("nq", [1, 3, 20])
@pytest.mark.parametrize("size", [2.0 ** 127, 2.0 ** 100, 2.0 ** -100, 2.0 ** -125])
def test_queries_of_every_finite_size(gen, kind, nq, size):
    """Queries near both ends of the type's range, the softmax scale bringing
    the scores back."""
    k, v = make(gen, 90, 2, 64, kind)
    small = 2.0 ** -6 if size > 1 else 2.0 ** 6
    q = (torch.randn(nq, 8, 64, generator=gen, device="cuda").clamp(-1.9, 1.9).double() * size).to(TYPES[kind])
    assert q.isfinite().all() and q.abs().amax() > size
    s = Setup(gen, kind, 90, nq, 2, 4, 64, (k.float() * small).to(TYPES[kind]), v, q, scale=0.1 / small / size)
    close(s.call(), s.want(), slice(None), kind)


def test_a_closed_cache_refuses_every_call(gen):
    from rustyllm_b200 import RqError
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.rope import qk_norm_rope_append, rope_tables
    cache = KV4Cache(1, 16, 2, 32)
    k, v = make(gen, 1, 2, 32, "f32")
    calls = (lambda: cache.append(k, v, i32(0)), lambda: cache.append(k[:0], v[:0], i32()), lambda: cache.read(i32(0)),
             lambda: cache.attention(k, i32(0)[None], i32(1)), lambda: cache.device_bytes(),
             lambda: qk_norm_rope_append(cache, k, k, v, i32(0), i32(0), *rope_tables(1, 32)))
    for call in calls:
        call()
    cache.close()
    cache.close()
    for call in calls:
        with pytest.raises(RqError, match="NULL"):
            call()


def test_scales_that_pass_f32_in_base_2_are_refused(gen):
    from rustyllm_b200 import RqError
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(1, 16, 1, 32)
    for scale in (3e38, -2.4e38, 1e39, math.nan):
        with pytest.raises(RqError, match="scale"):
            cache.attention(torch.zeros(1, 1, 32, device="cuda"), i32(0)[None], i32(1), scale=scale)
    assert not cache.attention(torch.zeros(1, 1, 32, device="cuda"), i32(0)[None], i32(1), scale=2.3e38).any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 21, 40])
@pytest.mark.parametrize("at", [3, 70])
def test_small_weights_count_beside_a_value_without_weight(gen, kind, nq, at):
    """Most of the weight on a position without value, the rest on 240 others
    at some 2^-18 of it, whose values make the output, and at `at` the largest
    value that the cache can hold, without weight.  (Short enough that no form
    splits the positions.)"""
    n = 240
    k, v = make(gen, n, 2, 64, kind)
    k, v = (k.float() * 0.05).to(TYPES[kind]), v.abs()
    q = torch.randn(nq, 8, 64, generator=gen, device="cuda").abs().to(TYPES[kind])
    k[100], v[100] = 2, 0
    k[at] = -20
    v[at] = 6e4 if kind == "f16" else 5.2e5
    s = Setup(gen, kind, n, nq, 2, 4, 64, k, v, q)
    close(s.call(), s.want(), slice(None), kind)
