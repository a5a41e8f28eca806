"""Cases of the serving operators: prompt attention, paged decode attention, rotary + cache append, sampling.

Each case is one call a serving loop makes.  Shapes are those of the two decoder shapes this repository ships
(7B: 32 query and 32 KV heads; 70B: 64 and 8; its tensor-parallel shard of eight: 8 and 1; head dimension 128), its
context lengths and batch sizes, and generic lengths around them.  With `own` false the operators run in elementary
torch operations in 32 bits (64 for the sampling, whose borders need it); with `own` true through asmllm_b200.ops.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a chat turn's first tokens on the 7B shape: launch latency and one short tile per head
        dict(name="prompt_short_7b", op="prompt", lens="33", prefix="0", nh=32, nkv=32, hd=128, dtype="fp16",
             out="fp16", page=0),
        # one long document on the 7B shape, keys and values packed like the queries
        dict(name="prompt_8192_7b", op="prompt", lens="8192", prefix="0", nh=32, nkv=32, hd=128, dtype="bf16",
             out="bf16", page=0),
        # a batch of prompts of different lengths on the 70B shape, read back from the cache they were appended to
        dict(name="prompt_ragged_70b", op="prompt",
             lens="1024,7,513,128,1,890,255,640,77,1000,300,129,450,961,36,702", prefix="0", nh=64, nkv=8, hd=128,
             dtype="bf16", out="bf16", page=16),
        # the next 512 tokens of four long prompts on one of eight tensor-parallel ranks (chunked prefill)
        dict(name="prompt_chunk_70b_tp8", op="prompt", lens="512,512,500,512", prefix="7680,4100,2047,15873", nh=8,
             nkv=1, hd=128, dtype="fp16", out="fp16", page=64),
        # batch-1 decode at the 7B shape's context length of 512
        dict(name="paged_one_7b", op="paged", batch=1, lo=512, hi=512, nh=32, nkv=32, hd=128, dtype="fp16",
             out="fp32", page=16),
        # the 70B shape's batch of 32 at different positions of a 1024-position context
        dict(name="paged_b32_70b", op="paged", batch=32, lo=1, hi=1024, nh=64, nkv=8, hd=128, dtype="fp16",
             out="fp32", page=16),
        # one very long sequence on one of eight tensor-parallel ranks: one KV head, only the length to split
        dict(name="paged_long_70b_tp8", op="paged", batch=1, lo=131071, hi=131071, nh=8, nkv=1, hd=128,
             dtype="bf16", out="bf16", page=64),
        # a full server: 64 sequences of up to 16k positions, the cache far larger than the last-level cache
        dict(name="paged_b64_16k_70b", op="paged", batch=64, lo=1, hi=16384, nh=64, nkv=8, hd=128, dtype="bf16",
             out="bf16", page=32),
        # one decode step of the 70B batch: rotate, round and append 32 rows
        dict(name="rope_b32_70b", op="rope", lens="", batch=32, hi=1024, nh=64, nkv=8, hd=128, src="fp32",
             dtype="fp16", page=16),
        # a whole 8192-token prompt of the 7B shape into the cache
        dict(name="rope_8192_7b", op="rope", lens="8192", batch=1, hi=8192, nh=32, nkv=32, hd=128, src="fp32",
             dtype="fp16", page=16),
        # one sequence's next token over the 32000-word vocabulary, the usual settings
        dict(name="sample_one", op="sample", batch=1, vocab=32000, dtype="fp32", temp=0.8, top_k=40, top_p=0.95,
             min_p=0.0, mix=False),
        # a full batch whose rows each have their own settings, over a larger vocabulary
        dict(name="sample_b128_mixed", op="sample", batch=128, vocab=128256, dtype="fp32", temp=1.0, top_k=0,
             top_p=0.9, min_p=0.05, mix=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "paged", "rope", "sample"])
    nkv, group = rng.choice([(1, 8), (8, 8), (32, 1), (4, 4), (2, 5), (8, 1), (3, 2)])
    heads = dict(nh=nkv * group, nkv=nkv, hd=rng.choice([128, 128, 64]), dtype=rng.choice(["fp16", "bf16"]))
    page = rng.choice([16, 32, 64, 128])
    if op == "prompt":
        page = rng.choice([0, 0, page])
        batch, top = rng.choice([(1, 8192 if nkv * group <= 32 else 4096), (4, 2048), (13, 700)])
        lens = [_log(rng, 1, top) for _ in range(batch)]
        prefix = [rng.choice([0, _log(rng, 1, top)]) if page and batch > 1 else 0 for _ in range(batch)]
        return dict(op=op, lens=",".join(map(str, lens)), prefix=",".join(map(str, prefix)), page=page,
                    out=heads["dtype"], **heads)
    if op == "paged":
        batch = _log(rng, 1, 64)
        hi = min(_log(rng, 16, 100000), 4 * 10**6 // (batch * nkv))
        return dict(op=op, batch=batch, lo=rng.choice([0, 1, hi]), hi=hi, page=page,
                    out=rng.choice([heads["dtype"], "fp32"]) if heads["dtype"] == "fp16" else "bf16", **heads)
    if op == "rope":
        if rng.random() < 0.5:
            return dict(op=op, lens="", batch=_log(rng, 1, 256), hi=_log(rng, 32, 4096), page=page,
                        src=rng.choice(["fp32", heads["dtype"]]), **heads)
        n = rng.choice([1, 2, 7])
        lens = [_log(rng, 1, 8000 // n) for _ in range(n)]
        return dict(op=op, lens=",".join(map(str, lens)), batch=len(lens), hi=max(lens), page=page,
                    src=rng.choice(["fp32", heads["dtype"]]), **heads)
    return dict(op=op, batch=_log(rng, 1, 128), vocab=_log(rng, 100, 131072), dtype=rng.choice(["fp32", "fp32", "bf16"]),
                temp=round(rng.uniform(0.3, 1.5), 3), top_k=rng.choice([0, _log(rng, 1, 1000)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                min_p=rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)]), mix=rng.random() < 0.3)


def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _lens(case):
    """(query lengths, cached lengths after this call) of a case, as host lists."""
    if case["op"] == "prompt":
        q = _ints(case["lens"])
        pre = _ints(case["prefix"])
        pre = pre * len(q) if len(pre) == 1 else pre
        return q, [a + b for a, b in zip(q, pre)]
    if case["op"] == "rope" and case["lens"]:
        q = _ints(case["lens"])
        return q, q
    r = torch.Generator().manual_seed(case["batch"] * 131 + case["hi"])  # lengths belong to the case
    lo = case.get("lo", 1)
    n = torch.randint(lo, case["hi"] + 1, (case["batch"],), generator=r)
    n[0] = case["hi"]
    return [1] * case["batch"], n.tolist()


# ------------------------------------------------------------------ inputs
def _pages(case, kv, g, fill=True):
    """Page pool (K, V) and the table of a batch whose pages were handed out in random order, as by a server."""
    page, nkv, hd, dt = case["page"], case["nkv"], case["hd"], DT[case["dtype"]]
    need = [max(1, -(-n // page)) for n in kv]
    total, width = sum(need), max(need)
    perm = torch.randperm(total, generator=g, device="cuda").int()
    start = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)
    col = torch.arange(width, device="cuda")
    table = perm[(start[:, None] + col).clamp_max(total - 1)]
    table = torch.where(col < torch.tensor(need, device="cuda")[:, None], table, torch.zeros_like(table)).contiguous()
    shape = (total, page, nkv, hd)
    if not fill:
        return torch.zeros(shape, dtype=dt, device="cuda"), torch.zeros(shape, dtype=dt, device="cuda"), table
    mk = lambda: torch.randn(shape, generator=g, device="cuda", dtype=dt)  # noqa: E731
    return mk(), mk(), table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    st = dict(case=case)
    if case["op"] == "sample":
        B, V = case["batch"], case["vocab"]
        # language-model-like rows: a long flat tail and a few words that stand out
        x = rand(B, V) * 2.0
        x += 6.0 * (torch.rand(B, V, generator=g, device="cuda") < 40.0 / V) * rand(B, V).abs()
        st["logits"] = x.to(DT[case["dtype"]])
        st["u"] = torch.rand(B, generator=g, device="cuda")
        full = lambda v, t: torch.full((B,), v, dtype=t, device="cuda")  # noqa: E731
        st["temperature"], st["top_p"] = full(case["temp"], torch.float32), full(case["top_p"], torch.float32)
        st["min_p"], st["top_k"] = full(case["min_p"], torch.float32), full(case["top_k"], torch.int32)
        if case["mix"]:  # every row its own: greedy ones, top-k ones, nucleus ones, unrestricted ones
            r = torch.arange(B, device="cuda")
            st["temperature"] = torch.where(r % 5 == 0, 0.0, st["temperature"] + 0.1 * (r % 4))
            st["top_k"] = torch.where(r % 3 == 1, 50 + r, st["top_k"]).int()
            st["top_p"] = torch.where(r % 4 == 3, 1.0, st["top_p"])
            st["min_p"] = torch.where(r % 2 == 1, 0.0, st["min_p"])
        return st
    q_len, kv = _lens(case)
    B, T, nh, nkv, hd = len(q_len), sum(q_len), case["nh"], case["nkv"], case["hd"]
    dt = DT[case["dtype"]]
    st["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    st["cu_q"] = torch.tensor([0] + q_len, device="cuda").cumsum(0).int()
    if case["op"] == "rope":
        st["qkv"] = rand(T, (nh + 2 * nkv) * hd).to(DT[case["src"]])
        ang = torch.arange(max(kv), device="cuda")[:, None].double() / 10000.0 ** (
            torch.arange(0, hd, 2, device="cuda").double() / hd)
        st["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        st["k"], st["v"], st["table"] = _pages(case, kv, g, fill=False)
        st["decode"] = not case["lens"]
        return st
    # scores of standard deviation 2: some keys matter, none is alone
    st["q"] = (rand(T, nh, hd) * 2.0).to(dt)
    if case["page"]:
        st["k"], st["v"], st["table"] = _pages(case, kv, g)
    else:
        st["k"], st["v"] = rand(T, nkv, hd).to(dt), rand(T, nkv, hd).to(dt)
    st["out"] = DT[case["out"]]
    st["max_q"], st["max_kv"] = max(q_len), max(kv)
    return st


# ------------------------------------------------------------------ plain forms
def _plain_attention(st):
    """Sequences padded to the longest: scores, mask, softmax and the weighted sum in 32 bits."""
    case, q = st["case"], st["q"]
    B, Lq, Lk = st["kv_len"].numel(), st["max_q"], st["max_kv"]
    nkv, hd, T = case["nkv"], case["hd"], q.shape[0]
    grp = case["nh"] // nkv
    cu = st["cu_q"].long() if case["op"] == "prompt" else torch.arange(B + 1, device="cuda")
    qn, kn = cu[1:] - cu[:-1], st["kv_len"].long()
    i, j = torch.arange(Lq, device="cuda"), torch.arange(Lk, device="cuda")
    Q = q[(cu[:-1, None] + i).clamp_max(T - 1)].float().view(B, Lq, nkv, grp, hd).permute(0, 2, 3, 1, 4)
    if case["page"]:
        pg = case["page"]
        rows = st["table"].long()[:, j // pg] * pg + j % pg
        K, V = st["k"].view(-1, nkv, hd)[rows], st["v"].view(-1, nkv, hd)[rows]
    else:
        rows = (cu[:-1, None] + j).clamp_max(T - 1)
        K, V = st["k"][rows], st["v"][rows]
    K, V = K.float().permute(0, 2, 3, 1), V.float().transpose(1, 2)
    S = torch.matmul(Q.reshape(B, nkv, grp * Lq, hd), K).view(B, nkv, grp, Lq, Lk).mul_(1.0 / math.sqrt(hd))
    keep = (j <= (kn - qn)[:, None, None] + i[:, None]) & (j < kn[:, None, None])
    S.masked_fill_(~keep[:, None, None], -math.inf)
    m = S.amax(-1, keepdim=True)
    P = S.sub_(m.masked_fill_(m == -math.inf, 0.0)).exp_()
    l = P.sum(-1, keepdim=True)
    O = torch.matmul(P.view(B, nkv, grp * Lq, Lk), V).view(B, nkv, grp, Lq, hd)
    O = O / l.masked_fill(l == 0, 1.0)
    t = torch.arange(T, device="cuda")
    s = torch.searchsorted(cu, t, right=True) - 1
    return O.permute(0, 3, 1, 2, 4)[s, t - cu[s]].reshape(T, case["nh"], hd).to(st["out"])


def _plain_rope(st):
    case, x = st["case"], st["qkv"].float()
    nh, nkv, hd, pg, dt = case["nh"], case["nkv"], case["hd"], case["page"], DT[case["dtype"]]
    T, cu = x.shape[0], st["cu_q"].long()
    t = torch.arange(T, device="cuda")
    s = torch.searchsorted(cu, t, right=True) - 1
    p = st["kv_len"].long()[s] - (cu[s + 1] - cu[s]) + t - cu[s]
    x = x.view(T, nh + 2 * nkv, hd)
    qk = x[:, :nh + nkv].unflatten(-1, (hd // 2, 2))
    c, d = st["rope"][p, None, :, 0], st["rope"][p, None, :, 1]
    qk = torch.stack([qk[..., 0] * c - qk[..., 1] * d, qk[..., 0] * d + qk[..., 1] * c], -1).flatten(-2)
    slot = st["table"].long()[s, p // pg] * pg + p % pg
    st["k"].view(-1, nkv, hd)[slot] = qk[:, nh:].to(dt)
    st["v"].view(-1, nkv, hd)[slot] = x[:, nh + nkv:].to(dt)
    return qk[:, :nh].to(dt), st["k"], st["v"]


def _plain_sample(st):
    x = st["logits"].double()
    B, V = x.shape
    T, u = st["temperature"].double(), st["u"].double()
    k = torch.where(st["top_k"] > 0, st["top_k"], V)[:, None]
    v, order = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    w = torch.exp((v - v[:, :1]) / T.masked_fill(T == 0, 1.0)[:, None])
    w = w * (torch.arange(V, device="cuda") < k)
    before = w.cumsum(-1) - w
    keep = (before < st["top_p"].double()[:, None] * w.sum(-1, keepdim=True)) & (w >= st["min_p"].double()[:, None])
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    cum = w.cumsum(-1)
    token = (cum > u[:, None] * cum[:, -1:]).int().argmax(-1)
    return torch.where(T == 0, order[:, 0], token).int()


# ------------------------------------------------------------------ the framework's calls
def _own(st):
    from asmllm_b200 import ops

    case = st["case"]
    if case["op"] == "sample":
        return ops.rows_sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                               top_p=st["top_p"], min_p=st["min_p"])
    if case["op"] == "rope":
        q = ops.rope_append(st["qkv"], st["rope"], st["kv_len"], st["table"], st["k"], st["v"], case["nh"],
                            cu_q=None if st["decode"] else st["cu_q"])
        return q, st["k"], st["v"]
    if case["op"] == "paged":
        return ops.attention_paged(st["q"], st["k"], st["v"], st["table"], st["kv_len"], out_dtype=st["out"])
    if case["page"]:
        return ops.attention_prompt(st["q"], st["k"], st["v"], st["cu_q"], kv_len=st["kv_len"],
                                    page_table=st["table"], out_dtype=st["out"])
    return ops.attention_prompt(st["q"], st["k"], st["v"], st["cu_q"], out_dtype=st["out"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return (_plain_sample if op == "sample" else _plain_rope if op == "rope" else _plain_attention)(state)


# ------------------------------------------------------------------ work and 64-bit values
def work(case):
    if case["op"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + case["batch"] * 24, "flops": 4 * n}
    q_len, kv = _lens(case)
    nh, nkv, hd, T = case["nh"], case["nkv"], case["hd"], sum(q_len)
    if case["op"] == "rope":
        n = T * (nh + 2 * nkv) * hd
        return {"bytes": n * ((4 if case["src"] == "fp32" else 2) + 2) + T * hd * 4, "flops": 3 * T * (nh + nkv) * hd}
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q_len, kv) if m)
    io = T * nh * hd * (2 + (4 if case["out"] == "fp32" else 2))
    return {"bytes": io + sum(kv) * nkv * hd * 4, "flops": 4 * pairs * nh * hd}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        got = []
        for b in range(case["batch"]):
            x, T = st["logits"][b].double(), float(st["temperature"][b].double())
            if T == 0:
                got.append(int((x == x.max()).nonzero()[0]))
                continue
            e = torch.exp((x - x.max()) / T)
            o = torch.argsort(-x, stable=True)
            k = int(st["top_k"][b])
            o = o[:k] if k > 0 else o
            m = e[o] / e[o].sum()
            n = int((m.cumsum(0) - m < float(st["top_p"][b].double())).sum())
            o = o[:max(1, n)]
            o = o[(e[o] >= float(st["min_p"][b].double())) | (e[o] == 1)]
            o = o.sort().values
            c = e[o].cumsum(0)
            got.append(int(o[int((c <= float(st["u"][b].double()) * c[-1]).sum())]))
        return torch.tensor(got, dtype=torch.int32)
    q_len, kv = _lens(case)
    nh, nkv, hd, pg = case["nh"], case["nkv"], case["hd"], case["page"]
    grp, first, outs = nh // nkv, 0, []
    if case["op"] == "rope":
        qs, K, V = [], st["k"].double(), st["v"].double()
        x = st["qkv"].double().view(-1, nh + 2 * nkv, hd)
        for s, (n, m) in enumerate(zip(q_len, kv)):
            rows = x[first:first + n]
            p = torch.arange(m - n, m, device="cuda")
            cs = torch.view_as_complex(st["rope"].double().contiguous())[p][:, None]
            z = torch.view_as_complex(rows[:, :nh + nkv].unflatten(-1, (hd // 2, 2)).contiguous()) * cs
            z = torch.view_as_real(z).flatten(-2)
            qs.append(z[:, :nh])
            page = st["table"][s].long()[p // pg]
            K[page, p % pg] = z[:, nh:]
            V[page, p % pg] = rows[:, nh + nkv:]
            first += n
        return torch.cat(qs), K, V
    for s, (n, m) in enumerate(zip(q_len, kv)):
        q = st["q"][first:first + n].double()
        if pg:
            pages = st["table"][s].long()[:max(1, -(-m // pg))]
            k, v = (st[c][pages].double().flatten(0, 1)[:m] for c in ("k", "v"))
        else:
            k, v = (st[c][first:first + n].double() for c in ("k", "v"))
        o = torch.zeros(n, nh, hd, dtype=torch.float64, device="cuda")
        if m:
            gone = torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None]
            for h in range(nh):
                a = (q[:, h] @ k[:, h // grp].T) * hd ** -0.5
                o[:, h] = torch.softmax(a.masked_fill(gone, -math.inf), -1) @ v[:, h // grp]
        outs.append(o)
        first += n
    return torch.cat(outs)
