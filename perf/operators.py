"""Cases of the operators that serve and score several sequences at once.

  store   rows of keys and values of a batch of sequences into a pool of pages
  paged   attention of each sequence's new tokens (one: a decode step) over its pages
  packed  causal attention over whole prompts that lie one behind the other, without a cache
  logprobs  log probabilities of given tokens, entropy and the most likely alternatives of rows of logits

`run` makes the plain form of a case from elementary torch operations, or, with `own` set, the call of
this repository's operator that a user makes.
"""
import math

import torch

own = False

_F = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a decode step of 64 chats: one new row for each
        dict(name="store_decode64", op="store", n_seq=64, new_max=1, ctx_min=1, ctx_max=512, n_kv=8, hd=128, page=64, type="f32"),
        # three long prompts that enter the cache
        dict(name="store_prompts", op="store", n_seq=3, new_max=6000, ctx_min=0, ctx_max=0, n_kv=8, hd=128, page=16, type="f32"),
        # one chat, one token: latency
        dict(name="decode1", op="paged", n_seq=1, n_new=1, chunks=1, ctx_min=700, ctx_max=700, n_head=32, n_kv=8, hd=128, page=64, window=0, softcap=0.0, type="f32"),
        # 64 chats of mixed lengths, one token each
        dict(name="decode64_ragged", op="paged", n_seq=64, n_new=1, chunks=64, ctx_min=17, ctx_max=8191, n_head=32, n_kv=8, hd=128, page=64, window=0, softcap=0.0, type="f16"),
        # two very long documents, one token each
        dict(name="decode2_long", op="paged", n_seq=2, n_new=1, chunks=2, ctx_min=100001, ctx_max=131071, n_head=32, n_kv=8, hd=128, page=128, window=0, softcap=0.0, type="f32"),
        # a prompt that enters in chunks, one of its later chunks
        dict(name="chunk512_at_12k", op="paged", n_seq=1, n_new=512, chunks=1, ctx_min=12288, ctx_max=12288, n_head=32, n_kv=8, hd=128, page=64, window=0, softcap=0.0, type="f32"),
        # one step of a server: a chunk of two prompts beside 14 chats, 7 query heads for each KV head, small pages
        dict(name="mixed16", op="paged", n_seq=16, n_new=333, chunks=2, ctx_min=250, ctx_max=5000, n_head=28, n_kv=4, hd=128, page=16, window=0, softcap=0.0, type="f16"),
        # one short question of a small model: latency
        dict(name="packed_short", op="packed", n_seq=1, len_min=37, len_max=37, n_head=4, n_kv=2, hd=64, window=0, softcap=0.0, type="f16"),
        # 16 prompts of mixed lengths, packed
        dict(name="packed16_ragged", op="packed", n_seq=16, len_min=65, len_max=2047, n_head=32, n_kv=8, hd=128, window=0, softcap=0.0, type="f16"),
        # one long prompt
        dict(name="packed_8k", op="packed", n_seq=1, len_min=8192, len_max=8192, n_head=32, n_kv=8, hd=128, window=0, softcap=0.0, type="bf16"),
        # the answer row of a decode step, with 20 alternatives
        dict(name="logprobs_row", op="logprobs", rows=1, vocab=151936, top_k=20, type="f32"),
        # the scores of a 512-token prompt, with five alternatives a token
        dict(name="logprobs_prompt", op="logprobs", rows=512, vocab=151936, top_k=5, type="f32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "paged", "paged", "packed", "packed", "logprobs"])
    if op == "logprobs":
        vocab = _log(rng, 300, 151936)
        return dict(op=op, rows=_log(rng, 1, 512), vocab=vocab, top_k=rng.choice([0, 1, 5, 20, 50]), type=rng.choice(["f32", "f16", "bf16"]))
    n_kv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 96, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "store":
        return dict(op=op, n_seq=_log(rng, 1, 64), new_max=_log(rng, 1, 250), ctx_min=0, ctx_max=_log(rng, 1, 512), n_kv=n_kv, hd=hd, page=page,
                    type=rng.choice(["f32", "f16"]))
    n_head = n_kv * rng.choice([1, 3, 4, 7, 8])
    window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
    softcap = rng.choice([0.0, 0.0, 0.0, 30.0])
    if op == "packed":
        longest = _log(rng, 1, 4096)
        n_seq = _log(rng, 1, max(1, min(32, (4096 * 8192) // (n_head * longest * longest // 8 + longest))))
        return dict(op=op, n_seq=n_seq, len_min=max(1, longest // 3), len_max=longest, n_head=n_head, n_kv=n_kv, hd=hd, window=window, softcap=softcap,
                    type=rng.choice(["f16", "bf16"]))
    n_new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 512)])
    ctx = _log(rng, 16, 32768)
    n_seq = _log(rng, 1, max(1, min(64, 2 ** 28 // (n_head * n_new * ctx), 2 ** 28 // (n_kv * hd * ctx))))
    return dict(op=op, n_seq=n_seq, n_new=n_new, chunks=rng.randint(1, n_seq), ctx_min=max(1, ctx // 5), ctx_max=ctx, n_head=n_head, n_kv=n_kv, hd=hd, page=page,
                window=window, softcap=softcap, type=rng.choice(["f32", "f16"]))


# ---- inputs -----------------------------------------------------------------------------------


def _spread(n, lo, hi):
    """n lengths from lo to hi, evenly spread in an order that mixes long and short."""
    if n == 1:
        return [hi]
    at = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    step = next(s for s in range(max(1, n * 5 // 8), 2 * n) if math.gcd(s, n) == 1)
    return [at[i * step % n] for i in range(n)]


def _plan(case):
    """(new tokens, whole length) of each sequence."""
    n = case["n_seq"]
    if case["op"] == "packed":
        new = _spread(n, case["len_min"], case["len_max"])
        return new, new
    if case["op"] == "store":
        new = _spread(n, (case["new_max"] + 1) // 2, case["new_max"])
    else:
        new = [case["n_new"] if i * case["chunks"] % n < case["chunks"] else 1 for i in range(n)]
    return new, [a + c for a, c in zip(new, _spread(n, case["ctx_min"], case["ctx_max"]))]


def _pairs(case, new, lens):
    """Attended (query, key) pairs of one head."""
    w, total = case["window"], 0
    for a, n in zip(new, lens):
        if w == 0 or w >= n:
            total += a * n - a * (a - 1) // 2
        else:
            total += sum(min(p + 1, w) for p in range(n - a, n))
    return total


def _rows_read(case, new, lens):
    """Rows of keys that some query attends."""
    w = case["window"]
    return sum(n if w == 0 else min(n, a + w - 1) for a, n in zip(new, lens))


_contexts = {}


def _context():
    """One context of the library for the program, on torch's current stream."""
    import rust_interference_engine_b200 as rie
    s = torch.cuda.current_stream()
    key = (s.device.index, s.cuda_stream)
    if key not in _contexts:
        _contexts[key] = rie.Context(s.device.index, s)
    return rie, _contexts[key]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"case": case}

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    T = _F[case["type"]]
    if case["op"] == "logprobs":
        rows, vocab, k = case["rows"], case["vocab"], case["top_k"]
        # logits of a language model: a broad body and a few tokens far above it
        x = normal(rows, vocab, scale=2.0)
        lift = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
        x.scatter_add_(1, lift, normal(rows, 24, scale=4.0).abs() + 4.0)
        st["logits"] = x.to(T)
        st["targets"] = lift[:, 0].to(torch.int32)
        st["out"] = dict(logprob=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
                         top_ids=torch.empty(rows, k, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(rows, k, device="cuda"))
        if own:
            st["rie"], st["ctx"] = _context()
        return st
    new, lens = _plan(case)
    n_kv, hd = case["n_kv"], case["hd"]
    cu = [0]
    for a in new:
        cu.append(cu[-1] + a)
    n_tok = cu[-1]
    st.update(new=new, lens=lens, n_tok=n_tok, cu=ints(cu))
    if case["op"] != "packed":
        # a pool with a few spare pages; each sequence's pages lie scattered over it
        ps = case["page"]
        need = [-(-n // ps) for n in lens]
        n_pages, width = sum(need) + 5, max(need)
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        first = [sum(need[:i]) for i in range(len(need))]
        at = ints(first)[:, None] + torch.arange(width, dtype=torch.int32, device="cuda")[None, :]
        st["pages"] = order[at.clamp(max=n_pages - 1).long()].contiguous()
        st["len"] = ints(lens)
        st["k_pool"] = normal(n_pages, n_kv, ps, hd, dtype=torch.float16)
        st["v_pool"] = normal(n_pages, n_kv, ps, hd, dtype=torch.float16)
        if own:
            rie, ctx = st["rie"], st["ctx"] = _context()
            st["cache"] = rie.PagedCache(ctx, n_kv, hd, ps, n_pages, k=st["k_pool"], v=st["v_pool"])
            st["batch"] = rie.SeqBatch(st["cu"], st["len"], st["pages"], n_tok, max_len=max(lens))
    elif own:
        st["rie"], st["ctx"] = _context()
    if case["op"] == "store":
        st["k"] = normal(n_tok, n_kv * hd, dtype=T)
        st["v"] = normal(n_tok, n_kv * hd, dtype=T)
        return st
    # queries come with the attention scale applied; scores then spread over a few units
    st["q"] = normal(n_tok, case["n_head"] * hd, scale=2.0 / math.sqrt(hd), dtype=T)
    if case["op"] == "packed":
        st["k"] = normal(n_tok, n_kv * hd, dtype=T)
        st["v"] = normal(n_tok, n_kv * hd, dtype=T)
    st["out"] = torch.empty_like(st["q"])
    return st


# ---- one pass ---------------------------------------------------------------------------------


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    case, rie, ctx = st["case"], st["rie"], st["ctx"]
    if case["op"] == "store":
        st["cache"].store(st["batch"], st["k"], st["v"])
        return [st["k_pool"], st["v_pool"]]
    if case["op"] == "paged":
        rie.paged_attention(ctx, st["cache"], st["batch"], st["q"], case["n_head"], st["out"], window=case["window"], softcap=case["softcap"])
        return st["out"]
    if case["op"] == "packed":
        rie.packed_attention(ctx, st["q"], st["k"], st["v"], st["cu"], case["n_head"], case["n_kv"], case["hd"], st["out"], window=case["window"],
                             softcap=case["softcap"], max_len=case["len_max"])
        return st["out"]
    o = st["out"]
    rie.logprobs(ctx, st["logits"], st["targets"], o["logprob"], o["entropy"], o["top_ids"], o["top_logprobs"])
    return o


def _places(st):
    """Sequence and position of each new token."""
    t = torch.arange(st["n_tok"], dtype=torch.int32, device="cuda")
    seq = torch.bucketize(t, st["cu"], right=True) - 1
    lens = st["len"] if "len" in st else st["cu"][1:] - st["cu"][:-1]
    return t, seq, lens[seq] - (st["cu"][seq + 1] - t), lens


def _run_plain(st):
    case = st["case"]
    if case["op"] == "logprobs":
        return _logprobs_plain(st)
    t, seq, pos, lens = _places(st)
    n_kv, hd = case["n_kv"], case["hd"]
    if case["op"] == "store":
        page = st["pages"][seq, pos // case["page"]].long()
        slot = (pos % case["page"]).long()
        st["k_pool"][page, :, slot] = st["k"].view(-1, n_kv, hd).to(torch.float16)
        st["v_pool"][page, :, slot] = st["v"].view(-1, n_kv, hd).to(torch.float16)
        return [st["k_pool"], st["v_pool"]]
    # every sequence padded to the longest: queries [seq, head, new, hd], keys [seq, kv head, len, hd]
    n_seq, G, far, most = case["n_seq"], case["n_head"] // n_kv, max(st["lens"]), max(st["new"])
    at = (t - st["cu"][seq]).long()
    q = torch.zeros(n_seq, most, n_kv, G, hd, device="cuda")
    q[seq, at] = st["q"].view(-1, n_kv, G, hd).float()
    if case["op"] == "packed":
        k, v = torch.zeros(2, n_seq, far, n_kv, hd, device="cuda")
        k[seq, at] = st["k"].view(-1, n_kv, hd).float()
        v[seq, at] = st["v"].view(-1, n_kv, hd).float()
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    else:
        k, v = (x[st["pages"].long()].transpose(1, 2).reshape(n_seq, n_kv, -1, hd)[:, :, :far].float() for x in (st["k_pool"], st["v_pool"]))
    s = q.permute(0, 2, 3, 1, 4).reshape(n_seq, n_kv, G * most, hd) @ k.transpose(2, 3)
    s = s.view(n_seq, n_kv, G, most, far)
    if case["softcap"] > 0:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    where = torch.full((n_seq, most), -1, dtype=torch.int32, device="cuda")
    where[seq, at] = pos.to(torch.int32)
    key = torch.arange(far, dtype=torch.int32, device="cuda")
    seen = key <= where[..., None]
    if case["window"] > 0:
        seen &= key > where[..., None] - case["window"]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    o = (p.view(n_seq, n_kv, G * most, far) @ v).view(n_seq, n_kv, G, most, hd)
    o = o / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4)[seq, at].reshape(st["n_tok"], -1).to(_F[case["type"]])


def _logprobs_plain(st):
    x = st["logits"].float() + 0.0  # -0 orders as +0
    k = st["case"]["top_k"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1, dtype=torch.float64)
    lse = m[:, 0] + torch.log(z)
    entropy = torch.log(z) - (e * d).sum(-1, dtype=torch.float64) / z
    logprob = x.gather(1, st["targets"][:, None].long())[:, 0] - lse
    # the largest first, ties to the lowest index: one whole number that orders by value, then index
    b = x.view(torch.int32).long()
    order = torch.where(b < 0, -1 - (b & 0x7FFFFFFF), b)
    index = torch.arange(x.shape[1], device="cuda")
    ids = torch.topk(order * (1 << 31) + ((1 << 31) - 1 - index), k, dim=-1).indices
    return dict(logprob=logprob.float(), entropy=entropy.float(), top_ids=ids.to(torch.int32), top_logprobs=(x.gather(1, ids) - lse[:, None]).float())


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    size = _SIZE[case["type"]]
    if case["op"] == "logprobs":
        rows, vocab, k = case["rows"], case["vocab"], case["top_k"]
        return {"bytes": rows * (vocab * size + 12 + 8 * k), "flops": rows * vocab * 5}
    new, lens = _plan(case)
    n_tok, row = sum(new), case["n_kv"] * case["hd"]
    if case["op"] == "store":
        return {"bytes": 2 * n_tok * row * (size + 2), "flops": 2 * n_tok * row}
    pairs = _pairs(case, new, lens)
    io = 2 * n_tok * case["n_head"] * case["hd"] * size
    return {"bytes": io + 2 * 2 * row * _rows_read(case, new, lens), "flops": 4 * case["n_head"] * case["hd"] * pairs}


# ---- the definition, in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        rows = [_exact_row(case, x, int(t)) for x, t in zip(st["logits"], st["targets"].tolist())]
        return {"logprob": torch.stack([r[0] for r in rows]), "entropy": torch.stack([r[1] for r in rows]), "top_ids": None,
                "top_logprobs": torch.stack([r[2] for r in rows])}
    if case["op"] == "store":
        k, v = st["k_pool"].double(), st["v_pool"].double()
        table, done = st["pages"].tolist(), 0
        for i, (a, n) in enumerate(zip(st["new"], st["lens"])):
            at = [(table[i][p // case["page"]], p % case["page"]) for p in range(n - a, n)]
            page, slot = torch.tensor(at, device="cuda").unbind(1)
            for pool, x in ((k, st["k"]), (v, st["v"])):
                pool[page, :, slot] = x[done:done + a].double().view(a, case["n_kv"], case["hd"])
            done += a
        return [k, v]
    hd, G = case["hd"], case["n_head"] // case["n_kv"]
    out = torch.empty(st["n_tok"], case["n_head"], hd, dtype=torch.float64, device="cuda")
    q = st["q"].view(-1, case["n_head"], hd)
    done = 0
    for i, (a, n) in enumerate(zip(st["new"], st["lens"])):
        pos = torch.arange(n - a, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hidden = (j > pos) | ((j <= pos - case["window"]) if case["window"] else (j > n))
        for h in range(case["n_kv"]):
            if case["op"] == "packed":
                k, v = (x[done:done + n, h * hd:(h + 1) * hd].double() for x in (st["k"], st["v"]))
            else:
                mine = st["pages"][i, :-(-n // case["page"])].long()
                k, v = (x[mine, h].reshape(-1, hd)[:n].double() for x in (st["k_pool"], st["v_pool"]))
            for r in range(h * G, (h + 1) * G):
                s = torch.mm(q[done:done + a, r].double(), k.t())
                if case["softcap"]:
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                s[hidden] = -math.inf
                out[done:done + a, r] = torch.softmax(s, 1) @ v
        done += a
    return out.view(st["n_tok"], -1)


def _exact_row(case, x, target):
    lp = torch.log_softmax(x.double(), 0)
    return lp[target], -(lp.exp() * lp).sum(), lp.sort(descending=True).values[:case["top_k"]]
