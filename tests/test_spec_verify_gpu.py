"""rq_spec_verify on the GPU against the rule in 64 bits (sums of the f32 /
f16 / bf16 probabilities are taken in f64 on both sides, so tokens compare for
equality)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def verify_ref(p, q, drafts, counts, u, r):
    B, n1, V = p.shape
    tokens, acc = np.full((B, n1), -1, np.int64), np.zeros(B, np.int64)
    mass = lambda x: np.where(x > 0, np.minimum(x, 3.402823466e38), 0.0)  # noqa: E731  (NaN > 0 is false)
    for b in range(B):
        n = min(max(int(counts[b]), 0), n1 - 1)
        i = 0
        while i < n:
            x = drafts[b, i]
            if not 0 <= x < V or not u[b, i] * (mass(q[b, i, x]) if q is not None else 1.0) < mass(p[b, i, x]):
                break
            tokens[b, i] = x
            i += 1
        acc[b] = i
        w = mass(p[b, i])
        if i < n:
            if q is not None:
                less = np.maximum(w - mass(q[b, i]), 0)
            else:
                less = w.copy()
                if 0 <= drafts[b, i] < V:
                    less[drafts[b, i]] = 0
            w = less if less.sum() > 0 else w
        if w.sum() > 0:
            c = np.cumsum(w)
            hit = np.nonzero((w > 0) & (c > min(max(r[b], 0.0), float(np.float32(0.99999994))) * c[-1]))[0]
            tokens[b, i] = hit[0] if len(hit) else np.nonzero(w > 0)[0][-1]
    return tokens, acc


def make(seed, B, n, V, kind, sharp=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = sharp * torch.randn(B, n + 1, V, generator=g, device="cuda")
    p = torch.softmax(logits, -1).to(TYPES[kind])
    q = torch.softmax(logits[:, :n] + 0.5 * torch.randn(B, n, V, generator=g, device="cuda"), -1)
    d = torch.multinomial(q.reshape(-1, V), 1, generator=g).reshape(B, n).to(torch.int32) if n else torch.zeros(B, 0, dtype=torch.int32, device="cuda")
    return p, q.to(TYPES[kind]), d, torch.rand(B, n, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")


def run(p, q, d, u, r, counts=None):
    from rustyllm_b200.spec import spec_verify
    tokens, acc = spec_verify(p, d, u, r, q=q, n_drafts=counts)
    wt, wa = verify_ref(p.double().cpu().numpy(), None if q is None else q.double().cpu().numpy(), d.cpu().numpy(),
                        [d.shape[1]] * p.shape[0] if counts is None else counts.tolist(), u.double().cpu().numpy(), r.double().cpu().numpy())
    assert np.array_equal(acc.cpu().numpy(), wa)
    assert np.array_equal(tokens.cpu().numpy(), wt)
    return tokens, acc


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,n,V", [(1, 4, 32000), (3, 1, 1), (5, 0, 777), (7, 3, 128), (4, 40, 129), (2, 5, 300001), (33, 2, 4099)])
def test_tokens_match_the_rule(rq_ctx, kind, B, n, V):
    p, q, d, u, r = make(B + n, B, n, V, kind)
    run(p, q, d, u, r)
    run(p, None, d, u, r)  # certain drafts
    counts = torch.randint(-1, n + 3, (B,), dtype=torch.int32, device="cuda")
    run(p, q, d, u, r, counts)


def test_large_group_runs_and_strided_rows(rq_ctx):
    """A vocabulary whose share of a CTA passes the sums kept in shared
    memory, and rows of a wider matrix."""
    V = 512 * 512 * 8 + 77
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.rand(2, 2, V + 5, generator=g, device="cuda")
    run(wide[:, :, 3:V + 3], None, torch.tensor([[V - 1], [5]], dtype=torch.int32, device="cuda"),
        torch.tensor([[2.0], [0.0]], device="cuda"), torch.tensor([0.37, 0.999], device="cuda"))


def test_borders_and_odd_inputs(rq_ctx):
    V = 4096
    p = torch.full((6, 2, V), 1.0 / V, device="cuda")  # exact sums: borders fall on r = j / V
    q = torch.full((6, 1, V), 1.0 / V, device="cuda")
    d = torch.tensor([[7], [7], [-1], [V], [9], [11]], dtype=torch.int32, device="cuda")
    u = torch.tensor([[0.5], [1.0], [0.0], [0.0], [math.nan], [0.0]], device="cuda")
    r = torch.tensor([0.25, 0.5, 0.0, 1.0, math.nan, 1.0 - 2.0 ** -24], device="cuda")
    run(p, q, d, u, torch.nan_to_num(r))  # p == q: the leftover has no mass, p itself is drawn from
    from rustyllm_b200.spec import spec_verify
    assert spec_verify(p, d, u, r, q=q)[0][4, 0] == 0  # an r that is not a number counts as 0
    p[0, 1] = 0.0
    p[1, 0], q[1, 0] = 0.0, 0.0
    p[5, 1, :] = 0.0
    p[5, 1, 3], p[5, 1, 9], p[5, 1, 50] = math.nan, -4.0, 1e-30
    tokens, acc = run(p, q, d, u, torch.nan_to_num(r))
    assert tokens[0].tolist() == [7, -1] and tokens[1].tolist() == [-1, -1] and tokens[5].tolist() == [11, 50]
    p[5, 1, 2000] = math.inf
    assert run(p, q, d, u, torch.nan_to_num(r))[0][5, 1] == 2000


def test_acceptance_rate_is_the_overlap(rq_ctx):
    """Over many drawn drafts the output is distributed as the target: the
    first token's frequencies match p within 5 standard deviations."""
    from rustyllm_b200.spec import spec_verify
    B, V = 20000, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    p1 = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    q1 = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    d = torch.multinomial(q1, B, replacement=True, generator=g).to(torch.int32)[:, None]
    tokens, acc = spec_verify(p1.expand(B, 2, V), d, torch.rand(B, 1, generator=g, device="cuda"),
                              torch.rand(B, generator=g, device="cuda"), q=q1.expand(B, 1, V))
    f = torch.bincount(tokens[:, 0].long(), minlength=V).double() / B
    sd = (p1.double() * (1 - p1.double()) / B).sqrt()
    assert ((f - p1.double()).abs() < 5 * sd).all()


def test_refusals(rq_ctx):
    from rustyllm_b200 import RqError
    from rustyllm_b200.spec import spec_verify
    p, q, d, u, r = make(1, 2, 3, 100, "f32")
    for call, msg in ((lambda: spec_verify(p.cpu(), d, u, r, q=q), "CUDA"), (lambda: spec_verify(p, d.long(), u, r, q=q), "drafts"),
                      (lambda: spec_verify(p, d, u, r, q=q[:, :2]), "q:"), (lambda: spec_verify(p, d, u.double(), r, q=q), "u:"),
                      (lambda: spec_verify(p, d, u, r, q=q.half()), "q:"), (lambda: spec_verify(p.double(), d, u, r), "float32"),
                      (lambda: spec_verify(p.transpose(1, 2), d, u, r), "contiguous")):
        with pytest.raises(RqError, match=msg):
            call()
