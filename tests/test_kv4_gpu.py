"""The 4-bit paged cache on the GPU: quantization, reading back, attention
over it, the norm and rotation pass, the page tables and the run of them
together, against plain implementations in 64 bits.

Tolerances.  The cache's values are exact (a code is the nearest multiple of
an f16 scale, decided without rounding), so append / read compare for equality
in f32 and to one rounding (half a step of the type: 2^-8 bf16, 2^-11 f16
relative) else.  Attention with f32 queries: queries and probabilities
enter the products as f16 hi + lo (22 bits), sums are f32; scores of the size
used here (|s| <= 32) carry at most 32 * 2^-23 absolute error from the f32 sum,
i.e. 4e-6 relative in a probability, so 2e-5 of the row's largest value holds
for the output.  16-bit queries are exact in f16 (bf16 after the row's power of
two; elements below 2^-14 of the row's largest lose at most 2^-25 of it).  f16
takes the same two parts of a probability as f32.  More than eight bf16 rows a kv
head take one part, for which the bound is made: their probabilities are rounded to f16 and multiplied by the value's scale in f16:
two roundings of 2^-11, so the sum of p_j v_j is off by at most (2 * 2^-11 +
2^-22) sum p_j |v_j|, to which the output's own rounding adds half a step of its
type times |o|, and the f32 parts above 2e-5 of sum p_j |v_j|; the tests take
the sum of p_j |v_j| from the reference ("reach").  More than 16 bf16 rows
a kv head take the form with rounded operands: there the second rounding
of 2^-11 is the value's, and the keys are rounded to f16 as well, which moves a
score by at most D = 2^-11 scale sum_d |q_d k_d| and so, since every weight and
their sum move by at most exp(+-D), the output by (exp(2 D) - 1) sum p_j |v_j|."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def quantize_ref(x):
    """Blocks of 32 of the last axis -> values held, in float64 (numpy)."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    at = np.abs(b).argmax(-1)
    m = np.take_along_axis(b, at[..., None], -1)
    with np.errstate(over="ignore"):
        d = np.clip(m / -8, -65504, 65504).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(d == 0, 8, np.clip(np.floor(b / np.where(d == 0, 1, d) + 8.5), 0, 15))
    return ((c - 8) * d).reshape(x.shape)


def make(g, n, kv, hd, kind):
    k = torch.randn(n, kv, hd, generator=g, device="cuda")
    v = torch.randn(n, kv, hd, generator=g, device="cuda") * 0.5
    return k.to(TYPES[kind]), v.to(TYPES[kind])


@pytest.fixture
def gen(rq_ctx):
    return torch.Generator(device="cuda").manual_seed(11)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,hd,page,n", [(1, 32, 16, 1), (2, 64, 16, 33), (3, 96, 48, 100), (8, 128, 64, 257)])
def test_append_and_read_hold_the_nearest_codes(gen, kind, kv, hd, page, n):
    from rustyllm_b200.kv4 import KV4Cache
    pages = (n + page - 1) // page + 1
    cache = KV4Cache(pages, page, kv, hd)
    k, v = make(gen, n, kv, hd, kind)
    # blocks where rounding decides: zeros, one sign, ties of both signs, tiny and huge values
    k[0] = 0
    v[n // 2, 0, :32] = torch.tensor([3.0, -3.0] * 16)
    v[n - 1, 0, :32] = torch.arange(32) * 2.0 ** -20
    if kind != "f16":
        k[n - 1, kv - 1, :32] = 1e9
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n].to(torch.int32)
    cache.append(k, v, slots)
    every = torch.arange(pages * page, dtype=torch.int32, device="cuda")
    rk, rv = cache.read(every)
    for got, x in ((rk, k), (rv, v)):
        want = np.zeros((pages * page, kv, hd))
        want[slots.cpu().numpy()] = quantize_ref(x.float().cpu().numpy())
        assert np.array_equal(got.cpu().numpy().astype(np.float64), want)
    for t in ("f16", "bf16"):
        hk, _ = cache.read(every, TYPES[t])
        assert torch.equal(hk, rk.to(TYPES[t]))


def test_append_skips_slots_outside_and_takes_strided_rows(gen):
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(4, 16, 2, 64)
    for off in (0, 1):  # 16-byte aligned rows, and rows that are not
        qkv = torch.randn(6, 5 * 64 + off, generator=gen, device="cuda")
        k = qkv[:, off:off + 128].unflatten(1, (2, 64))
        v = qkv[:, 128 + off:256 + off].unflatten(1, (2, 64))
        slots = torch.tensor([3, -1, 64, 2 ** 31 - 1, 40, 17], dtype=torch.int32, device="cuda")
        before = cache.read(torch.arange(64, dtype=torch.int32, device="cuda"))
        cache.append(k, v, slots)
        after = cache.read(torch.arange(64, dtype=torch.int32, device="cuda"))
        for b, a, x in zip(before, after, (k, v)):
            want = b.clone().double()
            for i, s in ((0, 3), (4, 40), (5, 17)):
                want[s] = torch.from_numpy(quantize_ref(x[i].cpu().numpy()))
            assert torch.equal(a.double(), want)
    outside = cache.read(torch.tensor([-5, 64], dtype=torch.int32, device="cuda"))
    assert not outside[0].any() and not outside[1].any()


def test_not_a_number_stays_in_its_block_and_infinities_saturate(gen):
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(1, 16, 1, 64)
    k = torch.randn(2, 1, 64, generator=gen, device="cuda")
    v = k.clone()
    k[0, 0, 5] = math.nan
    v[1, 0, 40] = -math.inf
    cache.append(k, v, torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    rk, rv = cache.read(torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    assert rk[0, 0, :32].isnan().all() and not rk[0, 0, 32:].isnan().any() and not rk[1].isnan().any()
    assert rv[1, 0, 40] == -8 * 65504.0 and rv.isfinite().all()


def attention_ref(q, kval, vval, table, page, kv_lens, cu, scale, window, n_pages):
    """float64, row by row; kval, vval [slots, kv, hd] float64.  Returns the
    outputs and, for the tolerance, sum p |v| of each and what rounded keys move."""
    n, H, hd = q.shape
    kv = kval.shape[1]
    out = np.full((n, H, hd), np.nan)
    reach, moved = out.copy(), np.zeros((n, H, 1))
    many = H // kv * int(np.diff(cu).max()) > 16
    for b in range(table.shape[0]):
        L, nq = max(int(kv_lens[b]), 0), int(cu[b + 1] - cu[b])
        for i in range(nq):
            if not 0 <= cu[b] + i < n:
                continue
            pos = L - nq + i
            js = [j for j in range(max(0, pos - window + 1 if window else 0), min(pos + 1, table.shape[1] * page))
                  if 0 <= table[b, j // page] < n_pages]
            if not js:
                out[cu[b] + i] = reach[cu[b] + i] = 0
                continue
            js = np.array(js)
            slots = table[b, js // page].astype(np.int64) * page + js % page
            for h in range(H):
                s = kval[slots, h // (H // kv)] @ q[cu[b] + i, h] * scale
                p = np.exp(s - s.max())
                out[cu[b] + i, h] = (p / p.sum()) @ vval[slots, h // (H // kv)]
                reach[cu[b] + i, h] = (p / p.sum()) @ np.abs(vval[slots, h // (H // kv)])
                if many:
                    d = 2.0 ** -11 * abs(scale) * (np.abs(kval[slots, h // (H // kv)]) @ np.abs(q[cu[b] + i, h]))
                    moved[cu[b] + i, h] = np.expm1(min(2 * d.max(), 100))
    return out, reach, moved


def fill(cache, gen, kind="f32"):
    n = cache.n_pages * cache.page_size
    k, v = make(gen, n, cache.n_kv_heads, cache.head_dim, kind)
    every = torch.arange(n, dtype=torch.int32, device="cuda")
    cache.append(k, v, every)
    rk, rv = cache.read(every)
    return rk.double().cpu().numpy(), rv.double().cpu().numpy()


def close(got, ref, rows, kind):
    """The rows (a slice or list) of the reference against got, row for row."""
    want, reach, moved = ref[0][rows], ref[1][rows], ref[2][rows]
    got = got.double().cpu().numpy()
    if kind == "f32":
        tol = 2e-5 * np.abs(want).max(-1, keepdims=True) + 1e-30
    else:
        tol = (2 * 2.0 ** -11 + 2.0 ** -22 + 2e-5 + moved) * reach + HALF_STEP[kind] * np.abs(want) + 2.0 ** -24
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,kv,hd,page,lens,qs,window", [
    (8, 2, 64, 16, [1], [1], 0),
    (8, 8, 32, 16, [17, 0, 1, 300], [1, 1, 1, 1], 0),
    (14, 2, 64, 32, [5, 700, 33], [1, 1, 1], 20),
    (16, 1, 96, 48, [128, 257], [1, 1], 0),
    (32, 8, 128, 64, [63, 64, 65, 1000], [1, 1, 1, 1], 0),
    (24, 8, 128, 16, [40, 9, 200], [5, 9, 1], 0),
    (8, 2, 64, 16, [130, 61, 7], [64, 61, 3], 33),
    (12, 12, 32, 128, [260, 90], [17, 33], 0),
    (28, 4, 96, 16, [3], [7], 0),
])
def test_attention_matches_the_formula(gen, kind, H, kv, hd, page, lens, qs, window):
    """Ragged lengths, single tokens and several, grouped heads of every
    count, pages that end inside a tile's reach, windows, and (last case) more
    queries than positions: the first see nothing."""
    from rustyllm_b200.kv4 import KV4Cache
    B, width = len(lens), max((max(lens) + page - 1) // page, 1) + 1
    cache = KV4Cache(B * width + 2, page, kv, hd)
    kval, vval = fill(cache, gen, kind)
    table = torch.randperm(B * width + 2, generator=gen, device="cuda")[:B * width].view(B, width).to(torch.int32)
    cu = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
    q = torch.randn(int(cu[-1]) + 2, H, hd, generator=gen, device="cuda").to(TYPES[kind])
    out = torch.full_like(q, 7.0)
    kl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = attention_ref(q.double().cpu().numpy(), kval, vval, table.cpu().numpy(), page, lens, cu, hd ** -0.5, window,
                         cache.n_pages)
    cache.attention(q, table, kl, cu_q=torch.from_numpy(cu).cuda(), max_q=max(qs), window=window, out=out)
    close(out[:cu[-1]], want, slice(0, cu[-1]), kind)
    assert (out[cu[-1]:] == 7).all()  # rows behind the last sequence
    if max(qs) == 1:
        close(cache.attention(q[:B], table, kl, window=window, max_len=max(lens)), want, slice(0, B), kind)
    # the output may be the query
    cache.attention(q, table, kl, cu_q=torch.from_numpy(cu).cuda(), max_q=max(qs), window=window, out=q)
    assert torch.equal(q[:cu[-1]], out[:cu[-1]])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("qn", [1, 4, 40])
def test_long_sequence_is_split_and_joined(gen, kind, qn):
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(320, 32, 2, 64)
    kval, vval = fill(cache, gen, kind)
    lens = [10007, 3]
    table = torch.randperm(320, generator=gen, device="cuda").to(torch.int32)
    table = torch.stack([table, table.flip(0)]).contiguous()
    cu = np.array([0, qn, 2 * qn], np.int32)
    q = torch.randn(2 * qn, 8, 64, generator=gen, device="cuda").to(TYPES[kind])
    want = attention_ref(q.double().cpu().numpy(), kval, vval, table.cpu().numpy(), 32, lens, cu, 0.3, 0, 320)
    got = cache.attention(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu_q=torch.from_numpy(cu).cuda(),
                          max_q=qn, scale=0.3)
    close(got, want, slice(None), kind)


def test_hidden_positions_do_not_enter(gen):
    """Not-a-number blocks behind a sequence's end, before its window and at
    positions that only later queries see; pages outside the cache."""
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(8, 16, 2, 64)
    kval, vval = fill(cache, gen)
    nan = torch.full((4, 2, 64), math.nan, device="cuda")
    # page 3 holds positions 32..47: 45.. lie behind the end (45), 44 is seen by the last query alone
    cache.append(nan, nan, torch.tensor([3 * 16 + 12, 3 * 16 + 13, 3 * 16 + 14, 3 * 16 + 15], dtype=torch.int32, device="cuda"))
    table = torch.tensor([[1, 0, 3, -1], [5, 99, 6, -7]], dtype=torch.int32, device="cuda")
    cu = np.array([0, 3, 4], np.int32)
    q = torch.randn(4, 8, 64, generator=gen, device="cuda")
    lens = [45, 60]
    out = cache.attention(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                          cu_q=torch.from_numpy(cu).cuda(), max_q=3)
    want = attention_ref(q.double().cpu().numpy(), kval, vval, table.cpu().numpy(), 16, lens, cu, 0.125, 0, 8)
    close(out[[0, 1, 3]], want, [0, 1, 3], "f32")
    assert out[2].isnan().all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("B,most_q,most", [(300, 1, 90), (150, 3, 40), (129, 1, 700)])
def test_batches_of_many_sequences(gen, kind, B, most_q, most):
    """More sequences than a CTA looks up at a time, of all lengths, some of
    them empty and some without queries; the pieces of the line begin and end
    anywhere."""
    from rustyllm_b200.kv4 import KV4Cache
    rng = np.random.default_rng(B)
    lens = rng.integers(0, most + 1, B)
    lens[rng.random(B) < 0.2] = 0
    lens[5] = 10 * most
    qs = np.ones(B, int) if most_q == 1 else rng.integers(0, most_q + 1, B)
    width = (10 * most + 15) // 16
    cache = KV4Cache(width + 40, 16, 2, 32)
    kval, vval = fill(cache, gen, kind)
    table = torch.randint(0, cache.n_pages, (B, width), generator=gen, device="cuda").to(torch.int32)
    cu = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
    q = torch.randn(int(cu[-1]), 8, 32, generator=gen, device="cuda").to(TYPES[kind])
    want = attention_ref(q.double().cpu().numpy(), kval, vval, table.cpu().numpy(), 16, lens, cu, 32 ** -0.5, 0, cache.n_pages)
    got = cache.attention(q, table, torch.from_numpy(lens.astype(np.int32)).cuda(),
                          cu_q=None if most_q == 1 else torch.from_numpy(cu).cuda(), max_q=most_q)
    close(got, want, slice(None), kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompts_over_missing_pages_and_odd_rows(gen, kind):
    """The many-rows form: pages outside the cache, not-a-number blocks that
    only later queries see, a query row that is not a number, and rows behind
    n_tokens."""
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(40, 16, 2, 64)
    kval, vval = fill(cache, gen, kind)
    cache.append(torch.full((1, 2, 64), math.nan, device="cuda"), torch.full((1, 2, 64), math.nan, device="cuda"),
                 torch.tensor([7 * 16 + 5], dtype=torch.int32, device="cuda"))
    table = torch.arange(1, 17, dtype=torch.int32, device="cuda")[None].repeat(2, 1)
    table[0, 3], table[0, 9], table[1, 0] = -1, 40, 2 ** 31 - 1
    at = 6 * 16 + 5  # page 7 is the table's entry 6: position 101
    lens, qs = [130, 75], [70, 75]
    cu = np.array([0, 70, 145], np.int32)
    q = torch.randn(145, 8, 64, generator=gen, device="cuda").to(TYPES[kind])
    q[80, 3] = math.nan   # position 10, on the absent page: sees nothing
    q[100, 3] = math.nan  # position 30
    want = attention_ref(q.double().cpu().numpy(), kval, vval, table.cpu().numpy(), 16, lens, cu, 0.125, 0, 40)
    out = torch.full_like(q, 5.0)
    cache.attention(q[:140], table, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu_q=torch.from_numpy(cu).cuda(),
                    max_q=75, out=out[:140])
    clean = [r for r in range(140) if not (r < 70 and lens[0] - 70 + r >= at) and r != 100]
    close(out[clean], want, clean, kind)
    assert out[[r for r in range(70) if lens[0] - 70 + r >= at]].isnan().all()
    assert not out[80].any() and out[100, 3].isnan().all() and not out[100, [0, 1, 2, 4, 5, 6, 7]].isnan().any()
    # and for single tokens
    one = cache.attention(q[100:101], table[1:], torch.tensor([31], dtype=torch.int32, device="cuda"))
    assert one[0, 3].isnan().all() and not one[0, [0, 1, 2, 4, 5, 6, 7]].isnan().any()
    assert (out[140:] == 5).all()


@pytest.mark.parametrize("kind,qn,ratio", [("f32", 1, 0), ("f32", 13, 0), ("f16", 2, 1.5), ("f16", 13, 1.5), ("bf16", 2, 1.5),
                                           ("bf16", 13, 1.5)])
def test_error_does_not_grow_with_the_walk(gen, kind, qn, ratio):
    """24000 positions of one kv head under 8 query heads.  f32: per tile of 16
    the products' cut-off sums lose at most 16 * 2^-23 of sum p |v|, hi + lo
    parts 2^-21, scores within 16 carry 16 * 2^-22 into the weights, and adding
    1500 tiles in f32 walks sqrt(1500) * 2^-25: 7e-6 of the output if all signs
    agreed, 2e-6 in the mean over rows and elements, whose signs are free.  16 bits:
    no more than 1.5 times what rounding the output alone leaves (bf16: three
    roundings of an eighth beside it, sqrt(1 + 3 / 64))."""
    from rustyllm_b200.kv4 import KV4Cache
    n = 24000
    cache = KV4Cache(n // 16, 16, 1, 64)
    k, v = make(gen, n, 1, 64, kind)
    every = torch.arange(n, dtype=torch.int32, device="cuda")
    cache.append(k, v, every)
    rk, rv = (x[:, 0].double() for x in cache.read(every))
    q = torch.randn(qn, 8, 64, generator=gen, device="cuda").to(TYPES[kind])
    got = cache.attention(q, every[:n // 16][None], torch.tensor([n], dtype=torch.int32, device="cuda"),
                          cu_q=torch.tensor([0, qn], dtype=torch.int32, device="cuda"), max_q=qn).double()
    s = q.double() @ rk.T * 64 ** -0.5
    s.masked_fill_(every > (n - qn + torch.arange(qn, device="cuda"))[:, None, None], -math.inf)
    want = s.softmax(-1) @ rv
    off = ((got - want).norm() / want.norm()).item()
    alone = ((want.to(TYPES[kind]).double() - want).norm() / want.norm()).item()
    assert off < (ratio * alone if ratio else 2e-6)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("H,kv,hd,page,lens,qs,window", [
    (8, 1, 32, 16, [300, 40, 0, 17], [30, 17, 0, 17], 0),
    (16, 2, 128, 64, [400, 257, 90], [40, 7, 16], 0),
    (32, 2, 96, 32, [1000, 129], [9, 128], 50),
    (16, 1, 128, 16, [2500], [20], 0),
    (7, 1, 64, 16, [500, 64, 65], [64, 64, 37], 0),
])
def test_prompts_of_more_than_one_tile_of_rows(gen, kind, H, kv, hd, page, lens, qs, window):
    """Row counts around one and two tiles of 128, steps that end inside a tile
    of positions, sequences without queries, one that is split."""
    from rustyllm_b200.kv4 import KV4Cache
    B, width = len(lens), (max(lens) + page - 1) // page
    cache = KV4Cache(B * width + 1, page, kv, hd)
    kval, vval = fill(cache, gen, kind)
    table = torch.randperm(B * width + 1, generator=gen, device="cuda")[:B * width].view(B, width).to(torch.int32)
    cu = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
    q = torch.randn(int(cu[-1]) + 3, H, hd, generator=gen, device="cuda").to(TYPES[kind])
    want = attention_ref(q.double().cpu().numpy(), kval, vval, table.cpu().numpy(), page, lens, cu, hd ** -0.5, window,
                         cache.n_pages)
    out = torch.full_like(q, 3.0)
    cache.attention(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu_q=torch.from_numpy(cu).cuda(),
                    max_q=max(qs), window=window, out=out)
    close(out[:cu[-1]], want, slice(0, cu[-1]), kind)
    assert (out[cu[-1]:] == 3).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [0.05, -0.05, 0.0])
@pytest.mark.parametrize("falls", [False, True])
def test_prompts_over_values_of_every_size(gen, kind, scale, falls):
    """The form with rounded operands: values that grow or fall by 10^6 over
    the sequence, and at its last position, which the last query alone sees,
    the cache's largest keys and values, 2^24 times their neighbours'.  (The
    scores stay within e^-4.4 of one another, so that no weight comes near the
    end of f16's range.)  Values that are not numbers in the last one's place
    leave the other queries within the same bounds."""
    from rustyllm_b200.kv4 import KV4Cache
    n, nq, kv, hd = 203, 101, 2, 96
    cache = KV4Cache(16, 16, kv, hd)
    k, v = make(gen, n, kv, hd, kind)
    k = (k.float() / k.float().abs().amax() * 4).to(TYPES[kind])
    size = torch.logspace(-2, 4, n, device="cuda")
    v = (v.float() / v.float().abs().amax(-1, keepdim=True) * (size.flip(0) if falls else size)[:, None, None]).to(TYPES[kind])
    k[-1] = v[-1] = 6e4 if kind == "f16" else 5e5
    slots = torch.arange(n, dtype=torch.int32, device="cuda") + 16
    cache.append(k, v, slots)
    every = torch.arange(256, dtype=torch.int32, device="cuda")
    rk, rv = cache.read(every)
    table = torch.arange(1, 16, dtype=torch.int32, device="cuda")[None]
    cu = np.array([0, nq], np.int32)
    q = torch.randn(nq, 8, hd, generator=gen, device="cuda").clamp(-4, 4).to(TYPES[kind])
    want = attention_ref(q.double().cpu().numpy(), rk.double().cpu().numpy(), rv.double().cpu().numpy(), table.cpu().numpy(),
                         16, [n], cu, scale, 0, 16)
    lens, cu = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.from_numpy(cu).cuda()
    got = cache.attention(q, table, lens, cu_q=cu, max_q=nq, scale=scale)
    close(got[:-1], want, slice(0, nq - 1), kind)
    v[-1] = math.nan
    cache.append(k, v, slots)
    again = cache.attention(q, table, lens, cu_q=cu, max_q=nq, scale=scale)
    close(again[:-1], want, slice(0, nq - 1), kind)


def test_slots_past_four_gigabytes(gen):
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(70000, 64, 8, 128)  # 5.2 GB
    assert cache.device_bytes() > 2 ** 32
    k, v = make(gen, 64, 8, 128, "f32")
    page = 69999
    slots = torch.arange(page * 64, page * 64 + 64, dtype=torch.int32, device="cuda")
    cache.append(k, v, slots)
    rk, rv = cache.read(slots)
    assert np.array_equal(rk.double().cpu().numpy(), quantize_ref(k.cpu().numpy()))
    low, _ = cache.read(torch.arange(0, 4096, dtype=torch.int32, device="cuda"))
    assert not low.any()
    q = torch.randn(1, 8, 128, generator=gen, device="cuda")
    table = torch.tensor([[page]], dtype=torch.int32, device="cuda")
    got = cache.attention(q, table, torch.tensor([64], dtype=torch.int32, device="cuda"))
    p = torch.softmax(torch.einsum("hd,jhd->hj", q[0].double(), rk.double()) / 128 ** 0.5, -1)
    want = torch.einsum("hj,jhd->hd", p, rv.double())
    assert ((got[0].double() - want).abs() <= 2e-5 * want.abs().amax(-1, keepdim=True)).all()


def test_calls_on_two_streams_and_in_two_graphs_do_not_meet(gen):
    """The same cache read by two streams at once, and by two captured graphs
    replayed at once: every call has its own workspace."""
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(600, 16, 2, 64)
    fill(cache, gen)
    lens = torch.tensor([9600], dtype=torch.int32, device="cuda")
    table = torch.randperm(600, generator=gen, device="cuda").to(torch.int32)[None].contiguous()
    qs = [torch.randn(1, 16, 64, generator=gen, device="cuda") for _ in range(2)]
    want = [cache.attention(q, table, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(20):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(cache.attention(q, table, lens))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for q, s in zip(qs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(cache.attention(q, table, lens))
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    del graphs


@pytest.mark.parametrize("scale_v", [2.0 ** -12, 1.0, 2.0 ** 10])
def test_f32_accuracy_does_not_depend_on_the_values_scale(gen, scale_v):
    """Values of any size: the probabilities' f16 parts are taken relative to
    the largest p * scale, so the error stays that of f32 sums."""
    from rustyllm_b200.kv4 import KV4Cache
    cache = KV4Cache(64, 16, 2, 128)
    k = torch.randn(1024, 2, 128, generator=gen, device="cuda")
    v = torch.randn(1024, 2, 128, generator=gen, device="cuda") * scale_v
    v[::7] *= 30.0
    every = torch.arange(1024, dtype=torch.int32, device="cuda")
    cache.append(k, v, every)
    rk, rv = cache.read(every)
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(1, 16, 128, generator=gen, device="cuda")
    want = attention_ref(q.double().cpu().numpy(), rk.double().cpu().numpy(), rv.double().cpu().numpy(), table.cpu().numpy(),
                         16, [1024], [0, 1], 128 ** -0.5, 0, 64)[0]
    got = cache.attention(q, table, torch.tensor([1024], dtype=torch.int32, device="cuda")).double().cpu().numpy()
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < 2e-6


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,kv,hd,rot,inter,norm,off", [
    (8, 2, 64, 64, False, True, 0), (5, 1, 128, 64, False, True, 0), (3, 3, 96, 96, True, False, 0),
    (4, 2, 256, 256, False, True, 0), (4, 2, 32, 16, True, True, 0), (2, 2, 80, 80, False, True, 0),
    (2, 1, 10, 6, False, True, 0), (2, 1, 10, 6, True, True, 0), (8, 2, 64, 64, False, True, 1), (4, 0, 64, 0, False, True, 0),
])
@pytest.mark.parametrize("n", [1, 37])
def test_norm_and_rotation_match_the_formula(gen, kind, H, kv, hd, rot, inter, norm, off, n):
    from rustyllm_b200.rope import qk_norm_rope, rope_tables
    flat = torch.randn(n, (H + 2 * kv) * hd + off, generator=gen, device="cuda").to(TYPES[kind])
    q = flat[:, off:off + H * hd].unflatten(1, (H, hd))
    k = flat[:, off + H * hd:off + (H + kv) * hd].unflatten(1, (kv, hd)) if kv else flat.new_empty(n, 0, hd)
    cos, sin = rope_tables(500, rot)
    pos = torch.randint(0, 500, (n,), generator=gen, device="cuda").to(torch.int32)
    if n > 1:
        pos[3], pos[5] = -1, 500  # padding, and behind the tables
    qw = 1 + 0.1 * torch.randn(hd, generator=gen, device="cuda") if norm else None
    kw = 1 + 0.1 * torch.randn(hd, generator=gen, device="cuda") if norm else None

    def ref(x, w):
        y = x.double()
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        p = pos.clamp(0, 499).long()
        c, s = cos.double()[p][:, None] if rot else None, sin.double()[p][:, None] if rot else None
        r = y.clone()
        if rot:
            i = torch.arange(0, rot, 2, device="cuda") if inter else torch.arange(rot // 2, device="cuda")
            j = i + (1 if inter else rot // 2)
            r[..., i], r[..., j] = y[..., i] * c - y[..., j] * s, y[..., i] * s + y[..., j] * c
        return r

    live = (pos >= 0) & (pos < 500) if rot else pos >= 0
    qo, ko = torch.full_like(q.contiguous(), 3.0), torch.full_like(k.contiguous(), 3.0)
    want = ref(q, qw), ref(k, kw)
    qk_norm_rope(q, k, pos, cos, sin, q_weight=qw, k_weight=kw, interleaved=inter, q_out=qo, k_out=ko)
    for got, w in zip((qo, ko), want):
        # f32 sums and one rounding of the result
        tol = (HALF_STEP[kind] + 8 * 2.0 ** -24) * w.abs() + 8 * 2.0 ** -24 * w.abs().amax(-1, keepdim=True).clamp(min=1e-6) if w.numel() else w
        assert ((got.double() - w).abs() <= tol)[live].all()
        assert (got[~live] == 3).all()
    # in place
    keep = flat.clone()
    qk_norm_rope(q, k, pos, cos, sin, q_weight=qw, k_weight=kw, interleaved=inter, q_out=q, k_out=k)
    assert torch.equal(q[live], qo[live]) and torch.equal(k[live], ko[live])
    assert torch.equal(flat[~live], keep[~live]) and torch.equal(flat[:, off + (H + kv) * hd:], keep[:, off + (H + kv) * hd:])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd,rot,inter,norm", [(64, 64, False, True), (96, 48, False, False), (128, 128, True, True), (32, 6, False, True)])
def test_rotation_with_append_equals_the_two_passes(gen, kind, hd, rot, inter, norm):
    """In one launch, k is quantized from the rotated f32 value; in two, from
    its rounding to k's type, so for f32 a code may differ only where the last
    bits of the rotation fall on a border (f32 sums in another order), and for
    16-bit types values may differ by a step of the block.  With h half a step
    of k's type, the two scales differ by (h + 2 * 2^-11) d at most (the
    rounding of the largest element, and of each scale to f16), x / d by less
    than one, so the codes by one at most, and the values |c1 d1 - c2 d2| <=
    |c1 - c2| d1 + 8 |d1 - d2| <= d (1 + 9 (h + 2^-10)).  Where two elements tie
    in magnitude and the scale's sign turns, an end is held as 8 d1 once and
    as 7 d2 the other time: the same bound."""
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.rope import qk_norm_rope, qk_norm_rope_append, rope_tables
    n, H, kv = 21, 6, 3
    q = torch.randn(n, H, hd, generator=gen, device="cuda").to(TYPES[kind])
    k, v = make(gen, n, kv, hd, kind)
    cos, sin = rope_tables(100, rot)
    pos = torch.randint(0, 100, (n,), generator=gen, device="cuda").to(torch.int32)
    slots = torch.randperm(64, generator=gen, device="cuda")[:n].to(torch.int32)
    pos[4], slots[7] = 100, -1
    w = dict(q_weight=torch.rand(hd, generator=gen, device="cuda") + 0.5, k_weight=torch.rand(hd, generator=gen, device="cuda") + 0.5) if norm else {}
    one, two = KV4Cache(4, 16, kv, hd), KV4Cache(4, 16, kv, hd)
    q1 = qk_norm_rope_append(one, q, k, v, pos, slots, cos, sin, interleaved=inter, q_out=torch.zeros_like(q), **w)
    q2, k2 = qk_norm_rope(q, k, pos, cos, sin, interleaved=inter, q_out=torch.zeros_like(q), k_out=torch.zeros_like(k), **w)
    alive = torch.where(pos < 100, slots, -1)
    two.append(k2, v, alive)
    tol = 2 * HALF_STEP[kind] + 2.0 ** -20
    assert ((q1.double() - q2.double()).abs() <= tol * q2.double().abs() + 1e-6).all()
    every = torch.arange(64, dtype=torch.int32, device="cuda")
    (a, b), (c, d) = one.read(every), two.read(every)
    assert torch.equal(b, d)
    step = c.unflatten(2, (-1, 32)).abs().amax(-1, keepdim=True) / 8
    off = (a - c).unflatten(2, (-1, 32)).abs()
    assert (off <= step * (1 + 9 * (HALF_STEP[kind] + 2.0 ** -10))).all()
    if kind == "f32":
        assert (off > step / 2).float().mean() < 1e-3


def pages_ref(ctx, new, table, ring, free, page, n_tokens):
    table, head, left, short = table.copy(), int(free[0]), int(free[1]), 0
    pos, slot, cu = [], [], [0]
    for b in range(len(ctx)):
        held, total = -(-ctx[b] // page), -(-(ctx[b] + new[b]) // page)
        for i in range(held, min(total, table.shape[1])):
            if left:
                table[b, i] = ring[head]
                head, left = (head + 1) % len(ring), left - 1
            else:
                table[b, i] = -1
                short += 1
        for p in range(ctx[b], ctx[b] + new[b]):
            pg = table[b, p // page] if p // page < table.shape[1] else -1
            pos.append(p)
            slot.append(pg * page + p % page if pg >= 0 else -1)
        cu.append(cu[-1] + new[b])
    pad = n_tokens - len(pos)
    return table, [head, left, short], cu, (pos + [-1] * pad)[:n_tokens], (slot + [-1] * pad)[:n_tokens]


@pytest.mark.parametrize("B,page,most,pool,n_tokens,seed", [
    (1, 16, 1, 4, 1, 0), (5, 16, 40, 200, 300, 1), (16, 64, 1, 64, 16, 2), (700, 16, 9, 3000, 9000, 3), (40, 32, 500, 4000, 30000, 4),
    (9, 16, 60, 12, 700, 5), (3, 1, 5, 100, 40, 6),
])
def test_pages_extend_and_release(rq_ctx, B, page, most, pool, n_tokens, seed):
    """Rings that wrap, too few pages (case 5), padding, more requests than a
    CTA's threads (case 3), several CTAs (case 4)."""
    from rustyllm_b200.pages import PageTable
    rng = np.random.default_rng(seed)
    width = 4 * most // page + 3
    t = PageTable(B, width, pool, page)
    ring = rng.permutation(pool).astype(np.int32)
    t.ring.copy_(torch.from_numpy(ring))
    head = int(rng.integers(0, pool))
    t.free.copy_(torch.tensor([head, pool, 0], dtype=torch.int32))
    table, free, lens = np.full((B, width), -1, np.int32), [head, pool, 0], [0] * B
    for step in range(3):
        new = rng.integers(0, most + 1, B).tolist()
        r = t.extend(torch.tensor(new, dtype=torch.int32, device="cuda"), n_tokens)
        table, free, cu, pos, slot = pages_ref(lens, new, table, ring, free, page, n_tokens)
        lens = [a + b for a, b in zip(lens, new)]
        assert np.array_equal(t.table.cpu().numpy(), table) and t.free.tolist() == free
        assert r.cu_new.tolist() == cu and t.lens.tolist() == lens
        assert r.positions.tolist() == pos and r.slots.tolist() == slot
        keep = [int(rng.integers(0, n + 1)) if rng.random() < 0.5 else n for n in lens]
        t.release(torch.tensor(keep, dtype=torch.int32, device="cuda"))
        for b in range(B):
            for i in range(-(-keep[b] // page), min(-(-lens[b] // page), width)):
                if table[b, i] >= 0:
                    ring[(free[0] + free[1]) % pool] = table[b, i]
                    free[1] += 1
                table[b, i] = -1
        lens = keep
        assert np.array_equal(t.table.cpu().numpy(), table) and t.free.tolist()[:2] == free[:2]
        at = [(free[0] + i) % pool for i in range(free[1])]
        assert np.array_equal(t.ring.cpu().numpy()[at], ring[at]) and t.lens.tolist() == lens


def test_tokens_behind_the_table_or_the_rows_get_no_slot(rq_ctx):
    from rustyllm_b200.pages import pages_extend
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    r = pages_extend(i32(0, 0), i32(40, 3), table, torch.arange(9, dtype=torch.int32, device="cuda"), i32(0, 9, 0), 16, 41)
    assert table.tolist() == [[0, 1], [2, -1]] and r.free.tolist() == [3, 6, 0] and r.cu_new.tolist() == [0, 40, 43]
    assert r.slots.tolist() == list(range(32)) + [-1] * 8 + [32] and r.positions.tolist() == list(range(40)) + [0]
    r = pages_extend(i32(-4, 5), i32(-1, -7), table, torch.arange(9, dtype=torch.int32, device="cuda"), i32(3, 6, 0), 16, 2)
    assert r.kv_lens.tolist() == [0, 5] and r.slots.tolist() == [-1, -1] and r.free.tolist() == [3, 6, 0]


def test_a_serving_loop_runs_captured(gen):
    """Lengths -> pages, slots and positions -> norm, rotation and append ->
    attention, for prompts and then single tokens, the decode step replayed
    from one CUDA graph with device-side lengths; outputs equal a contiguous
    f64 implementation over the values that the cache holds."""
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.pages import PageTable
    from rustyllm_b200.rope import qk_norm_rope_append, rope_tables
    B, H, kv, hd, page = 3, 8, 2, 64, 16
    cache, pages = KV4Cache(24, page, kv, hd), PageTable(B, 8, 24, page)
    cos, sin = rope_tables(128, hd)
    w = torch.rand(hd, generator=gen, device="cuda") + 0.5
    prompts = [17, 1, 32]
    n = sum(prompts)
    qkv = torch.randn(n + 2, H + 2 * kv, hd, generator=gen, device="cuda")
    new = torch.tensor(prompts, dtype=torch.int32, device="cuda")

    def step(qkv, new, max_q):
        r = pages.extend(new, qkv.shape[0])
        q = torch.empty(qkv.shape[0], H, hd, device="cuda")
        qk_norm_rope_append(cache, qkv[:, :H], qkv[:, H:H + kv], qkv[:, H + kv:], r.positions, r.slots, cos, sin,
                            q_weight=w, k_weight=w, q_out=q)
        return q, cache.attention(q, pages.table, pages.lens, cu_q=r.cu_new, max_q=max_q)

    def check_step(q, out, lens, counts):
        every = torch.arange(24 * page, dtype=torch.int32, device="cuda")
        rk, rv = cache.read(every)
        cu = np.concatenate([[0], np.cumsum(counts)])
        want = attention_ref(q.double().cpu().numpy(), rk.double().cpu().numpy(), rv.double().cpu().numpy(),
                             pages.table.cpu().numpy(), page, lens, cu, hd ** -0.5, 0, 24)
        close(out[:cu[-1]], want, slice(0, cu[-1]), "f32")

    check_step(*step(qkv, new, 32), prompts, prompts)
    ones = torch.ones(B, dtype=torch.int32, device="cuda")
    x = torch.randn(B, H + 2 * kv, hd, generator=gen, device="cuda")
    check_step(*step(x, ones, 1), [18, 2, 33], [1, 1, 1])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        q, out = step(x, ones, 1)
    lens = [18, 2, 33]
    for _ in range(20):
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        graph.replay()
        lens = [n + 1 for n in lens]
        check_step(q, out, lens, [1, 1, 1])
    assert pages.lens.tolist() == lens
    pages.release(torch.tensor([0, 5, 0], dtype=torch.int32, device="cuda"))
    assert pages.free.tolist()[1:] == [23, 0] and pages.table[1].tolist()[1:] == [-1] * 7
    del graph


def test_refusals(gen):
    from rustyllm_b200 import RqError
    from rustyllm_b200.kv4 import KV4Cache
    for args, msg in (((0, 16, 1, 64), "pages"), ((1, 24, 1, 64), "multiple of 16"), ((1, 16, 1, 80), "head_dim 80"),
                      ((2 ** 27, 16, 1, 64), "2\\^31")):
        with pytest.raises(RqError, match=msg):
            KV4Cache(*args)
    cache = KV4Cache(2, 16, 2, 64)
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    for call, msg in (
            (lambda: cache.append(k, k[:2], slots), "differ"), (lambda: cache.append(k, k, slots.long()), "int32"),
            (lambda: cache.append(k.double(), k.double(), slots), "float32"), (lambda: cache.append(k.cpu(), k, slots), "cuda"),
            (lambda: cache.append(k[..., ::2], k, slots), "64"), (lambda: cache.read(slots.cpu()), "int32"),
            (lambda: cache.attention(torch.zeros(1, 3, 64, device="cuda"), table, one), "3 query heads"),
            (lambda: cache.attention(torch.zeros(1, 2, 64, device="cuda"), table.long(), one), "block_table"),
            (lambda: cache.attention(torch.zeros(0, 2, 64, device="cuda"), table, one), "0 tokens"),
            (lambda: cache.attention(torch.zeros(1, 2, 64, device="cuda"), table, one, window=-1), "window"),
            (lambda: cache.attention(torch.zeros(1, 2, 64, device="cuda"), table, one, scale=math.nan), "scale")):
        with pytest.raises(RqError, match=msg):
            call()
    import ctypes

    from rustyllm_b200 import _lib
    host = np.zeros(64, np.float32)
    pair = (ctypes.c_int64 * 2)(128, 64)
    assert _lib.lib().rq_kv4_append(cache.handle, 0, host.ctypes.data, pair, k.data_ptr(), pair, slots.data_ptr(), 1, None) == 1
    assert "k must be device memory" in _lib.last_error()


def test_refuses_outputs_whose_rows_lie_on_one_another_and_sizes_past_32_bits(gen):
    from rustyllm_b200 import RqError
    from rustyllm_b200.kv4 import KV4Cache
    from rustyllm_b200.pages import pages_extend, pages_release
    from rustyllm_b200.rope import qk_norm_rope, rope_tables
    cache = KV4Cache(2, 16, 2, 64)
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    two = torch.ones(2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 64, device="cuda")
    with pytest.raises(RqError, match="lie on one another"):
        cache.attention(q, table, two, out=torch.zeros(1, 4, 64, device="cuda").expand(2, 4, 64))
    with pytest.raises(RqError, match="lie on one another"):
        qk_norm_rope(q, q, two, *rope_tables(4, 64), q_out=torch.zeros(2, 1, 64, device="cuda").expand(2, 4, 64))
    ring, free = torch.arange(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 4, 0], dtype=torch.int32, device="cuda")
    with pytest.raises(RqError, match="out of range"):
        pages_extend(two, two, table, ring, free, 2 ** 32 + 16, 2)
    with pytest.raises(RqError, match="out of range"):
        pages_release(two, two, table, ring, free, 2 ** 32 + 16)
