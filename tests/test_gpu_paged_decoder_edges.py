"""PagedDecoder: which batch a step runs in, and the options that a model may have."""
import dataclasses

import numpy as np
import pytest
import torch

import paged_ref
from oracle.llama import LlamaRef, rms_norm, rope
from test_gpu_decode import _oracle_weights, _tiny
from test_gpu_paged_decoder import TOL

pytestmark = pytest.mark.gpu


def model(seed=7, **kw):
    from odiengine_b200.decode import seeded_model

    cfg = dataclasses.replace(_tiny(1), **kw)
    return cfg, seeded_model(cfg, seed=seed, interleave_gate_up=False)


@pytest.mark.parametrize("temperature", [None, 0.9])
@pytest.mark.parametrize("max_drafts", [7, 0])
def test_single_tokens_run_in_a_batch_of_single_tokens(cuda_lib, monkeypatch, temperature, max_drafts):
    """The batch's max_new chooses attention's kernel: one of drafts for single tokens of
    eight heads per kv head would be one for 64 rows with 8 in use.  Whatever the
    batch, a request's logits are those of its own sequence."""
    from odiengine_b200 import paged

    cfg, mw = model(heads=8, kv_heads=1)
    W = _oracle_weights(cuda_lib, cfg, mw)
    used = []
    real = paged.attention_paged
    monkeypatch.setattr(paged, "attention_paged", lambda q, c, t, b, *a, **kw: (used.append(b.max_new), real(q, c, t, b, *a, **kw))[1])
    g = torch.Generator(device="cuda").manual_seed(1)
    d = paged.PagedDecoder(cfg, mw, requests=3, num_pages=12, max_drafts=max_drafts, chunk=6, temperature=temperature, generator=g)
    ids = [d.add(p) for p in ([3, 4, 5], [9], [7, 8])]
    d.step()
    assert set(used) == {6, 1}  # two prompts in a chunk, the other's first token
    while any(d.left(b) for b in ids):
        d.step()
    refs = {b: (LlamaRef(cfg, W), []) for b in ids}
    fed = {0: [3, 4], 1: [9], 2: [7]}
    for b in ids:  # what is in the cache so far
        ref, toks = refs[b]
        assert d._len[b] == len(fed[b])
        for i, t in enumerate(fed[b]):
            ref.step(t, i)
        toks += fed[b]
    for drafts in ({}, {0: [1, 2], 2: [5]}, {}, {1: [6] * 7}, {}):
        drafts = {b: x[:max_drafts] for b, x in drafts.items()}
        used.clear()
        pending = {b: d._todo[b][0] for b in ids}
        out = d.step(drafts)
        assert set(used) == {1 + max_drafts if any(drafts.values()) else 1}
        lists, row, starts = {}, 0, [0]
        for b in ids:
            ref, toks = refs[b]
            lists[b] = [pending[b], *drafts.get(b, ())]
            want = np.stack([ref.step(t, len(toks) + i) for i, t in enumerate(lists[b])])
            got = d.logits[row:row + len(want)].cpu().numpy().astype(np.float64)
            assert np.abs(got - want).max() <= TOL[torch.float16] * np.abs(want).max()
            row += len(want)
            starts.append(row)
        logits, rows = d.logits[:row].cpu().numpy(), [t for b in ids for t in lists[b]]
        if temperature:
            acc, nxt = paged_ref.verify(logits, rows, starts, d.u_accept.tolist(), d.u_next.tolist(), temperature)
        for i, b in enumerate(ids):
            if not temperature:
                best = logits[starts[i]:starts[i + 1]].argmax(1)
                kept = next(k for k in range(len(best)) if k + 1 == len(best) or best[k] != lists[b][k + 1])
                assert out[b] == [*lists[b][1:1 + kept], best[kept]]
            else:
                assert out[b] == [*lists[b][1:1 + acc[i]], nxt[i]]
            refs[b][1].extend(lists[b][:len(out[b])])
    assert d.status() == 0


class OptionsRef(LlamaRef):
    """LlamaRef with capped scores and distance biases; rows of the cache in its type."""

    def __init__(self, cfg, W, softcap, slopes, dtype):
        super().__init__(cfg, W)
        self.softcap, self.slopes, self.dtype = softcap, slopes, dtype

    def cached(self, x):
        return torch.from_numpy(x).to(self.dtype).double().numpy()

    def step(self, token, pos):
        cfg, W = self.cfg, self.W
        H, KV, hd, F = cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.ffn
        x = W["token_embd"][token].astype(np.float64)
        for layer in range(cfg.layers):
            qkv = W[f"wqkv.{layer}"] @ rms_norm(x, W[f"attn_norm.{layer}"], cfg.eps)
            q, k, v = (qkv[a * hd:b * hd].reshape(-1, hd).copy() for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
            rope(q, pos, cfg.theta)
            rope(k, pos, cfg.theta)
            self.kc[layer, :, pos], self.vc[layer, :, pos] = self.cached(k), self.cached(v)
            att = np.zeros((H, hd))
            for h in range(H):
                s = self.kc[layer, h * KV // H, :pos + 1] @ q[h] / np.sqrt(hd)
                if self.softcap:
                    s = self.softcap * np.tanh(s / self.softcap)
                s = s - self.slopes[h] * np.arange(pos, -1, -1)
                p = np.exp(s - s.max())
                att[h] = p / p.sum() @ self.vc[layer, h * KV // H, :pos + 1]
            x = x + W[f"wo.{layer}"] @ att.reshape(-1)
            gu = W[f"wgu.{layer}"] @ rms_norm(x, W[f"ffn_norm.{layer}"], cfg.eps)
            g, u = gu[:F], gu[F:]
            x = x + W[f"wdown.{layer}"] @ (g / (1.0 + np.exp(-g)) * u)
        return W["output"] @ rms_norm(x, W["out_norm"], cfg.eps)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("softcap,biased", [(0.3, False), (0.0, True), (0.5, True)])
def test_capped_scores_and_distance_biases(cuda_lib, dtype, softcap, biased):
    """Both come after the rotation; prompts in chunks, single tokens and drafts.  The
    norms' weights are tripled, so that scores are about as large as the caps."""
    from odiengine_b200.paged import PagedDecoder

    cfg, mw = model(seed=11)
    for lw in mw.layers:
        lw.attn_norm.mul_(3)
    slopes = 2.0 ** -np.arange(1, cfg.heads + 1, dtype=np.float64) if biased else np.zeros(cfg.heads)
    refs = [OptionsRef(cfg, _oracle_weights(cuda_lib, cfg, mw), softcap, slopes, dtype) for _ in range(2)]
    plain = LlamaRef(cfg, refs[0].W)
    d = PagedDecoder(cfg, mw, requests=2, num_pages=8, dtype=dtype, max_drafts=3, chunk=20, softcap=softcap,
                     slopes=torch.tensor(slopes, dtype=torch.float32, device="cuda") if biased else None)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, cfg.vocab, n).tolist() for n in (30, 4)]
    for p in prompts:
        d.add(p)
    while d.left(0) or d.left(1):
        d.step()
    toks = [p[:-1] for p in prompts]
    for b in range(2):
        assert d._len[b] == len(toks[b])
        for i, t in enumerate(toks[b]):
            refs[b].step(t, i)
            if b == 0:
                plain.step(t, i)
    for drafts in ({}, {0: [5, 6, 7], 1: [8]}):
        fed = [[d._todo[b][0], *drafts.get(b, ())] for b in range(2)]
        out, row = d.step(drafts), 0
        for b in range(2):
            want = np.stack([refs[b].step(t, len(toks[b]) + i) for i, t in enumerate(fed[b])])
            got = d.logits[row:row + len(fed[b])].cpu().numpy().astype(np.float64)
            row += len(fed[b])
            assert np.abs(got - want).max() <= TOL[dtype] * np.abs(want).max(), np.abs(got - want).max() / np.abs(want).max()
            if b == 0 and not drafts:  # the options do something
                other = plain.step(fed[0][0], len(toks[0]))
                assert np.abs(other - want[0]).max() > 3 * TOL[dtype] * np.abs(want).max()
            toks[b] = toks[b] + fed[b][:len(out[b])]
    assert d.status() == 0
