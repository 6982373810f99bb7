"""A run of the operators together, as a program that serves several sequences uses them next to
the framework's matmuls: prompts in one packed call, their keys and values into pages, decode steps
over the pages, scores of the answers. One attention layer with Q8_0 weights, checked against the
same layer computed sequence by sequence in 64 bits from the weights' own values."""
import numpy as np
import pytest

import oracle as O

pytestmark = pytest.mark.gpu

N_EMBD, N_HEAD, N_KV, HD, VOCAB, PS = 256, 4, 2, 64, 640, 16


@pytest.fixture(scope="module")
def layer():
    import torch
    import rust_interference_engine_b200 as rie
    ctx = rie.Context(0, torch.cuda.current_stream())
    rng = O.Rng(99)
    shapes = dict(q=(N_HEAD * HD, N_EMBD), k=(N_KV * HD, N_EMBD), v=(N_KV * HD, N_EMBD), o=(VOCAB, N_HEAD * HD))
    w = {n: rie.Weight.upload(ctx, rie.GgmlType.Q8_0, r, c, rng.weight(O.Q8_0, r, c)) for n, (r, c) in shapes.items()}
    return torch, rie, ctx, w


def project(layer, x, names, outs):
    torch, rie, ctx, w = layer
    acts = rie.QuantActs(ctx, x.shape[0], x.shape[1])
    acts.prepare(x, x.shape[0], x.shape[1], rie.ActFormat.Q8_0)
    rie.matmul_multi(ctx, acts, [rie.MatmulJob(w[n], o, o.shape[1]) for n, o in zip(names, outs)])


def exact_attention(q, k, v, first):
    """q rows at positions first.. over k, v (64 bits; k and v as the cache holds them)."""
    out = np.zeros_like(q)
    for t in range(q.shape[0]):
        for h in range(N_HEAD):
            kk, vv = (x[:first + t + 1].reshape(-1, N_KV, HD)[:, h // (N_HEAD // N_KV)] for x in (k, v))
            s = kk @ q[t, h * HD:(h + 1) * HD]
            p = np.exp(s - s.max())
            out[t, h * HD:(h + 1) * HD] = p @ vv / p.sum()
    return out


def test_prompts_then_decode_then_scores(layer):
    torch, rie, ctx, w = layer
    g = torch.Generator(device="cuda").manual_seed(5)
    prompts, steps = [37, 1, 90], 3
    n_seq = len(prompts)
    cache = rie.PagedCache(ctx, N_KV, HD, PS, 32)
    pages = torch.randperm(32, generator=g, device="cuda")[:n_seq * 8].to(torch.int32).reshape(n_seq, 8).contiguous()
    ks = [np.zeros((0, N_KV * HD)) for _ in prompts]
    vs = [np.zeros((0, N_KV * HD)) for _ in prompts]
    lens = [0] * n_seq
    for step in range(1 + steps):
        new = prompts if step == 0 else [1] * n_seq
        n = sum(new)
        cu_h = np.concatenate([[0], np.cumsum(new)])
        lens = [a + b for a, b in zip(lens, new)]
        cu = torch.tensor(cu_h, dtype=torch.int32, device="cuda")
        batch = rie.SeqBatch(cu, torch.tensor(lens, dtype=torch.int32, device="cuda"), pages, n)
        x = torch.randn(n, N_EMBD, generator=g, device="cuda")
        q, k, v = (torch.zeros(n, h * HD, device="cuda") for h in (N_HEAD, N_KV, N_KV))
        project(layer, x, "qkv", (q, k, v))
        q *= HD ** -0.5 / 4
        cache.store(batch, k, v)
        att = torch.zeros_like(q)
        rie.paged_attention(ctx, cache, batch, q, N_HEAD, att)
        if step == 0:  # the same prompts without the cache
            packed = torch.zeros_like(q)
            rie.packed_attention(ctx, q, k.half(), v.half(), cu, N_HEAD, N_KV, HD, packed)
        logits = torch.zeros(n, VOCAB, device="cuda")
        project(layer, att, "o", (logits,))
        targets = torch.randint(0, VOCAB, (n,), generator=g, device="cuda").to(torch.int32)
        lp, ent = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        ids, top = torch.zeros(n, 7, dtype=torch.int32, device="cuda"), torch.zeros(n, 7, device="cuda")
        rie.logprobs(ctx, logits, targets, lp, ent, ids, top)
        ctx.sync()
        qn, kn, vn = q.double().cpu().numpy(), k.half().double().cpu().numpy(), v.half().double().cpu().numpy()
        for i in range(n_seq):
            a, b = cu_h[i], cu_h[i + 1]
            ks[i], vs[i] = np.concatenate([ks[i], kn[a:b]]), np.concatenate([vs[i], vn[a:b]])
            want = exact_attention(qn[a:b], ks[i], vs[i], lens[i] - new[i])
            # f32 sums of values below max |v| = V: scores off by 2^-20 |q| |k| at most, values by 2^-20 V
            V = np.abs(vs[i]).max()
            score = 2.0 ** -19 * np.linalg.norm(qn[a:b].reshape(-1, HD), axis=1).max() * np.linalg.norm(ks[i].reshape(-1, HD), axis=1).max()
            tol = (score + 2.0 ** -19) * V
            assert np.abs(att[a:b].double().cpu().numpy() - want).max() <= tol
            if step == 0:
                assert np.abs(packed[a:b].double().cpu().numpy() - want).max() <= tol
        y = logits.double().cpu().numpy()
        d = y - y.max(axis=1, keepdims=True)
        want = d - np.log(np.exp(d).sum(axis=1, keepdims=True))
        rows = np.arange(n)
        assert np.abs(lp.cpu().numpy() - want[rows, targets.cpu().numpy()]).max() <= 2.0 ** -17 * (1 + np.abs(want).max())
        assert np.abs(ent.cpu().numpy() + (np.exp(want) * want).sum(axis=1)).max() <= 2.0 ** -16 * np.log(VOCAB)
        assert (np.take_along_axis(y, ids.cpu().numpy().astype(int), axis=1) == -np.sort(-y, axis=1)[:, :7]).all()
        assert np.abs(top.cpu().numpy() - np.take_along_axis(want, ids.cpu().numpy().astype(int), axis=1)).max() <= 2.0 ** -17 * (1 + np.abs(want).max())
