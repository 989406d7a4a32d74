"""The Llama loop with its cache in 4 bits and pages, and with q/k norms.

The reference model below runs in float64 over the dequantized weights, but
attends over the keys and values that the model's cache holds, so it differs
from the model by the arithmetic of the linears alone (relative L2 1e-4, the
loop's own bar) and not by which of two codes a key on a border got.  The
cache itself is checked against the reference's keys and values: a held value
is within half a step of its block, a whole step at the end that 4 bits clip,
plus what the linears' error moves."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(hidden=512, intermediate=1024, n_heads=8, n_kv_heads=2, head_dim=64, n_layers=2, vocab=1000, max_seq=100,
           max_batch_tokens=32, rms_eps=1e-5, rope_theta=10000.0)
TOL = 2e-4  # logits, relative L2: one bar of the linears for the model, one for what the cache's keys carry


def build(seed, cfg=CFG, norm=False, page=16, kv4=True):
    from rustyllm_b200.llama import random_model
    model, host = random_model(cfg, 12, seed, host_tensors=True)
    if kv4:
        model.use_kv4(page)
    rng = np.random.default_rng(seed)
    norms = []
    for l in range(cfg["n_layers"]):
        w = [(1 + 0.2 * rng.standard_normal(cfg["head_dim"])).astype(np.float32) for _ in range(2)] if norm else None
        if norm:
            model.set_qk_norm(l, *w)
        norms.append(w)
    return model, host, norms


class Ref:
    def __init__(self, model, host, norms, cfg, held):
        self.cfg, self.norms, self.host, self.model, self.held = cfg, norms, host, model, held
        self.w = [[torch.from_numpy(w.dequantize()).double() for w in model.layer_weights(l)] for l in range(cfg["n_layers"])]
        self.k = [np.zeros((0, cfg["n_kv_heads"], cfg["head_dim"])) for _ in range(cfg["n_layers"])]
        self.v = [x.copy() for x in self.k]

    def rms(self, x, w, eps):
        return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * torch.from_numpy(np.asarray(w)).double()

    def rotate(self, x, pos):
        hd = self.cfg["head_dim"]
        inv = 1.0 / np.float32(self.cfg["rope_theta"]) ** (np.arange(0, hd, 2, dtype=np.float32) / np.float32(hd))
        a = torch.from_numpy(pos.astype(np.float32)[:, None] * inv.astype(np.float32)).double()[:, None]
        f, g = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat((f * a.cos() - g * a.sin(), f * a.sin() + g * a.cos()), -1)

    def forward(self, tokens, pos0):
        """Logits at every position; call after the model has run the tokens."""
        c = self.cfg
        T, nh, nkv, hd, eps = len(tokens), c["n_heads"], c["n_kv_heads"], c["head_dim"], c["rms_eps"]
        x = torch.from_numpy(self.host["embed"][np.asarray(tokens)].astype(np.float64))
        pos = np.arange(pos0, pos0 + T)
        for l in range(c["n_layers"]):
            _, r1, r2 = self.host["layers"][l]
            w = self.w[l]
            h = self.rms(x, r1, eps)
            q, k, v = (h @ w[i].T for i in range(3))
            q, k, v = q.view(T, nh, hd), k.view(T, nkv, hd), v.view(T, nkv, hd)
            if self.norms[l]:
                q, k = self.rms(q, self.norms[l][0], eps), self.rms(k, self.norms[l][1], eps)
            q, k = self.rotate(q, pos), self.rotate(k, pos)
            if self.held:
                hk, hv = (torch.from_numpy(a).double() for a in self.model.read_kv4(l, 0, pos0 + T))
                for got, want in ((hk[pos0:], k), (hv[pos0:], v)):
                    b = want.reshape(T, nkv, -1, 32)
                    step = b.abs().amax(-1, keepdim=True) / 8
                    assert ((got.reshape(b.shape) - b).abs() <= step * (1 + 2.0 ** -9) + 8e-3 * step * 8).all()
                    # off the clipped end half a step holds; the linears' error allowed as above
                    inner = b.abs() < 7 * step
                    assert ((got.reshape(b.shape) - b).abs() <= step * (0.5 + 2.0 ** -8 + 8e-3 * 8))[inner].all()
            else:
                self.k[l] = np.concatenate((self.k[l][:pos0], k.numpy()))
                self.v[l] = np.concatenate((self.v[l][:pos0], v.numpy()))
                hk, hv = torch.from_numpy(self.k[l]), torch.from_numpy(self.v[l])
            g = nh // nkv
            s = torch.einsum("thd,jhd->htj", q, hk.repeat_interleave(g, 1)) / hd ** 0.5
            s = s.masked_fill(torch.arange(pos0 + T)[None, None] > torch.from_numpy(pos)[None, :, None], -np.inf)
            a = torch.einsum("htj,jhd->thd", torch.softmax(s, -1), hv.repeat_interleave(g, 1)).reshape(T, nh * hd)
            x = x + a @ w[3].T
            h = self.rms(x, r2, eps)
            u = h @ w[4].T
            x = x + (u * torch.sigmoid(u) * (h @ w[5].T)) @ w[6].T
        return (self.rms(x, self.host["ln_f"], eps) @ torch.from_numpy(self.host["lm_head"].astype(np.float64)).T).numpy()


def rel(a, b):
    return float(np.linalg.norm(np.asarray(a, np.float64) - b) / np.linalg.norm(b))


@pytest.mark.parametrize("kv4,norm,page,hd", [(True, False, 16, 64), (True, True, 32, 64), (False, True, 0, 64), (True, True, 16, 128)])
def test_logits_of_prompts_steps_and_verification(rq_ctx, kv4, norm, page, hd):
    cfg = dict(CFG, head_dim=hd, n_heads=512 // hd)
    model, host, norms = build(3, cfg, norm, page, kv4)
    ref = Ref(model, host, norms, cfg, kv4)
    rng = np.random.default_rng(1)
    pos = 0
    for T in (19, 1, 3, 26, 1, 5):  # prompts, single tokens, verification widths
        ids = rng.integers(0, cfg["vocab"], T).astype(np.int32)
        logits, amax = model.forward_all(ids, pos, want_logits=True)
        want = ref.forward(ids, pos)
        assert rel(logits, want) <= TOL
        pos += T
    # roll back into the middle of a page and go on with other tokens
    model.truncate_caches(21)
    ids = rng.integers(0, cfg["vocab"], 9).astype(np.int32)
    logits, _ = model.forward(ids, 21)
    assert rel(logits, ref.forward(ids, 21)[-1]) <= TOL
    model.close()


def test_decode_steps_replayed_from_a_graph(rq_ctx):
    """generate (device-side steps that take pages as they go) equals forwards
    of one token each, and a captured step replayed equals both; fused steps
    fall back to the launch chain."""
    model, _, _ = build(5, norm=True)
    prompt = np.random.default_rng(2).integers(0, CFG["vocab"], 14).astype(np.int32)
    want = model.generate(prompt, 40)
    model.set_fused(True)
    assert model.generate(prompt, 40) == want
    model.set_fused(False)
    _, tok = model.forward(prompt, 0, want_logits=False)
    seq = [tok]
    for i in range(39):
        _, tok = model.forward([tok], len(prompt) + i, want_logits=False)
        seq.append(tok)
    assert seq == want
    from rustyllm_b200._lib import check, lib
    check(lib().rq_llama_reset_tokens(model.handle))
    model.forward(prompt, 0, want_logits=False)
    model.decode_step()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        model.decode_step(torch.cuda.current_stream().cuda_stream)
    for _ in range(38):
        graph.replay()
    torch.cuda.synchronize()
    toks, pos = model.tokens()
    assert toks[:40] == want and pos == 14 + 39
    del graph
    model.close()


def test_steps_past_the_capacity_do_no_harm(rq_ctx):
    model, _, _ = build(6, dict(CFG, max_seq=40))
    model.forward(np.arange(30, dtype=np.int32), 0, want_logits=False)
    for _ in range(30):
        model.decode_step()
    torch.cuda.synchronize()
    model.status()
    model.truncate_caches(30)
    a, _ = model.forward([7], 30)
    model.truncate_caches(30)
    b, _ = model.forward([7], 30)
    assert np.array_equal(a, b) and np.isfinite(a).all()
    model.close()


def test_refusals(rq_ctx):
    from rustyllm_b200 import RqError
    from rustyllm_b200.llama import random_model
    model, _ = random_model(dict(CFG, n_layers=1, head_dim=16, n_heads=32), 12, 1)
    with pytest.raises(RqError, match="head_dim 16"):
        model.use_kv4(16)
    assert model.forward([1, 2], 0)[0].shape == (1000,)  # still works on the f32 cache
    with pytest.raises(RqError, match="f32"):
        model.read_kv4(0, 0, 1)
    with pytest.raises(RqError, match="expected 16"):
        model.set_qk_norm(0, np.ones(8), np.ones(16))
    model.close()
    model, _ = random_model(dict(CFG, n_layers=1), 12, 1)
    with pytest.raises(RqError, match="multiple of 16"):
        model.use_kv4(20)
    model.use_kv4(16)
    with pytest.raises(RqError, match="already"):
        model.use_kv4(16)
    with pytest.raises(RqError, match="positions"):
        model.read_kv4(0, 99, 2)
    model.close()


def test_sampled_speculation_follows_the_rule(rq_ctx, monkeypatch):
    """The sampled loop: every verification's tokens follow from its inputs by
    the rule, the same seed gives the same tokens, a draft equal to the target
    is accepted, and it runs on the 4-bit cache."""
    import rustyllm_b200.spec as spec
    from tests.test_spec_verify_gpu import verify_ref
    target, _, _ = build(71)
    draft, _, _ = build(72, kv4=False)
    prompt = np.random.default_rng(3).integers(0, CFG["vocab"], 10).astype(np.int32)
    real, seen = spec.spec_verify, []

    def watched(p, drafts, u, r, q=None, n_drafts=None):
        out = real(p, drafts, u, r, q=q, n_drafts=n_drafts)
        wt, wa = verify_ref(p.double().cpu().numpy(), None if q is None else q.double().cpu().numpy(), drafts.cpu().numpy(),
                            [drafts.shape[1]], u.double().cpu().numpy(), r.double().cpu().numpy())
        assert np.array_equal(out[0].cpu().numpy(), wt) and out[1].tolist() == wa.tolist()
        assert (p.sum(-1) - 1).abs().max() < 1e-4
        seen.append(drafts.shape[1])
        return out

    monkeypatch.setattr(spec, "spec_verify", watched)
    runs = [spec.SpecDecoder(target, draft, k=3, temperature=0.8, seed=s).generate(prompt, 25) for s in (4, 4, 5)]
    assert runs[0] == runs[1] != runs[2] and all(len(r) == 25 and all(0 <= t < CFG["vocab"] for t in r) for r in runs)
    assert set(seen) == {0, 3}
    twin, _, _ = build(71)
    sd = spec.SpecDecoder(target, twin, k=4, temperature=0.8, adaptive=True)
    sd.generate(prompt, 40)
    assert sd.stats["accepted"] >= 0.9 * sd.stats["proposed"]
    for m in (target, draft, twin):
        m.close()
