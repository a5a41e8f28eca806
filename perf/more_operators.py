"""Cases of the serving operators around an 8-bit cache, a shared prefix and the logits before sampling.

  store    rotary append into a paged Q8_0 cache (8-bit codes, an fp16 scale for each block of 32 values), then rows
           of it read back in 16 bits for the prompt attention
  paged8   attention of one new token per sequence over that cache
  shared   attention of one new token per sequence where groups of sequences have the same first pages, which are
           read once for the whole group
  adjust   repetition, frequency and presence penalties, sparse biases and a bit mask of allowed words on logits

Shapes are those of the two decoder shapes this repository ships (7B: 32 query and 32 KV heads; 70B: 64 and 8; its
tensor-parallel shard of eight: 8 and 1; head dimension 128), its context lengths, batch sizes and vocabularies, and
generic lengths around them.  With `own` false the operators run in elementary torch operations in 32 bits; with
`own` true through asmllm_b200.ops.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of the 70B batch: rotate, quantise and append 32 rows; what was written, read back
        dict(name="store_b32_70b", op="store", lens="", prefix="", batch=32, hi=1024, nh=64, nkv=8, hd=128, src="fp32",
             dtype="fp16", page=16, whole=False),
        # a whole 8192-token prompt of the 7B shape into the cache, read back for its own attention
        dict(name="store_8192_7b", op="store", lens="8192", prefix="0", batch=1, hi=8192, nh=32, nkv=32, hd=128,
             src="fp32", dtype="fp16", page=16, whole=True),
        # the next 512 tokens of four long prompts of the 70B shape: appended, then all that each prompt holds read back
        dict(name="store_chunk_70b", op="store", lens="512,512,500,512", prefix="7680,4100,2047,15873", batch=4,
             hi=16385, nh=64, nkv=8, hd=128, src="bf16", dtype="bf16", page=64, whole=True),
        # batch-1 decode at the 7B shape's context length of 512
        dict(name="paged8_one_7b", op="paged8", batch=1, lo=512, hi=512, nh=32, nkv=32, hd=128, dtype="fp16",
             out="fp32", page=16),
        # the 70B shape's batch of 32 at different positions of a 1024-position context
        dict(name="paged8_b32_70b", op="paged8", batch=32, lo=1, hi=1024, nh=64, nkv=8, hd=128, dtype="fp16",
             out="fp32", page=16),
        # a full server: 64 sequences of up to 16k positions, the cache far larger than the last-level cache
        dict(name="paged8_b64_16k_70b", op="paged8", batch=64, lo=1, hi=16384, nh=64, nkv=8, hd=128, dtype="bf16",
             out="bf16", page=32),
        # eight chats on one system prompt of 1024 tokens, on one of eight tensor-parallel ranks
        dict(name="shared_b8_70b_tp8", op="shared", rows="8", shared="1024", lo=1, hi=128, nh=8, nkv=1, hd=128,
             dtype="fp16", out="fp16", page=16),
        # three prompts sampled several times over on the 7B shape, groups and prompts of different sizes
        dict(name="shared_groups_7b", op="shared", rows="16,5,27", shared="4096,1008,336", lo=1, hi=300, nh=32, nkv=32,
             hd=128, dtype="fp16", out="fp32", page=16),
        # a server whose 256 sequences continue one long document on the 70B shape
        dict(name="shared_b256_32k_70b", op="shared", rows="256", shared="32768", lo=1, hi=1024, nh=64, nkv=8, hd=128,
             dtype="bf16", out="bf16", page=64),
        # one sequence's logits with a repetition penalty over 512 tokens and a few biased words
        dict(name="adjust_one", op="adjust", batch=1, vocab=32000, dtype="fp32", hist=512, bias=8, mask=False),
        # a full batch over a larger vocabulary: long histories, biases and a grammar's mask
        dict(name="adjust_b128_mask", op="adjust", batch=128, vocab=128256, dtype="fp32", hist=8192, bias=64,
             mask=True),
        # 16-bit logits of a middle-sized batch
        dict(name="adjust_b32_bf16", op="adjust", batch=32, vocab=128256, dtype="bf16", hist=1024, bias=300,
             mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "paged8", "shared", "adjust"])
    nkv, group = rng.choice([(1, 8), (8, 8), (32, 1), (4, 4), (2, 5), (8, 1), (3, 2)])
    heads = dict(nh=nkv * group, nkv=nkv, hd=rng.choice([128, 128, 64]), dtype=rng.choice(["fp16", "bf16"]))
    page = rng.choice([16, 32, 64, 128])
    if op == "store":
        src = rng.choice(["fp32", heads["dtype"]])
        if rng.random() < 0.4:
            return dict(op=op, lens="", prefix="", batch=_log(rng, 1, 256), hi=_log(rng, 32, 4096), page=page, src=src,
                        whole=False, **heads)
        n = rng.choice([1, 2, 7])
        lens = [_log(rng, 1, 8000 // n) for _ in range(n)]
        whole = rng.random() < 0.7
        prefix = [_log(rng, 1, 8000 // n) if whole and n > 1 else 0 for _ in range(n)]
        return dict(op=op, lens=",".join(map(str, lens)), prefix=",".join(map(str, prefix)), batch=n,
                    hi=max(a + b for a, b in zip(lens, prefix)), page=page, src=src, whole=whole, **heads)
    if op == "paged8":
        batch = _log(rng, 1, 64)
        hi = min(_log(rng, 16, 100000), 4 * 10**6 // (batch * nkv))
        return dict(op=op, batch=batch, lo=rng.choice([0, 1, hi]), hi=hi, page=page,
                    out=rng.choice([heads["dtype"], "fp32"]), **heads)
    if op == "shared":
        n = rng.choice([1, 1, 2, 5])
        rows = [_log(rng, 1, 200 // n) for _ in range(n)]
        top = min(32768, 2 * 10**6 // nkv // n)
        shared = [max(1, _log(rng, 64, top) // page) * page for _ in range(n)]
        hi = min(_log(rng, 1, 2000), 10**6 // (nkv * sum(rows)))
        return dict(op=op, rows=",".join(map(str, rows)), shared=",".join(map(str, shared)), lo=1, hi=hi, page=page,
                    out=rng.choice([heads["dtype"], "fp32"]) if heads["dtype"] == "fp16" else "bf16", **heads)
    return dict(op=op, batch=_log(rng, 1, 128), vocab=_log(rng, 100, 131072), dtype=rng.choice(["fp32", "fp32", "bf16"]),
                hist=_log(rng, 1, 8192), bias=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.4)


def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _between(case, batch):
    """Lengths from lo to hi that belong to the case; the first is hi."""
    r = torch.Generator().manual_seed(batch * 131 + case["hi"])
    n = torch.randint(case.get("lo", 1), case["hi"] + 1, (batch,), generator=r)
    n[0] = case["hi"]
    return n.tolist()


def _lens(case):
    """(rows of this call, positions held after it, positions shared with the group) of each sequence."""
    if case["op"] == "shared":
        first = [p for n, p in zip(_ints(case["rows"]), _ints(case["shared"])) for _ in range(n)]
        return [1] * len(first), [a + b for a, b in zip(first, _between(case, len(first)))], first
    if case["op"] == "store" and case["lens"]:
        q, pre = _ints(case["lens"]), _ints(case["prefix"])
        return q, [a + b for a, b in zip(q, pre)], [0] * len(q)
    return [1] * case["batch"], _between(case, case["batch"]), [0] * case["batch"]


# ------------------------------------------------------------------ inputs
def _blocks(x):
    """Q8_0 of x [..., n] as this framework has it: codes int8 [..., n] and scales [..., n / 32] in fp16."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    inv = torch.where(top == 0, 0.0, 127.0 / top)
    return (b * inv).round_().clamp_(-128.0, 127.0).to(torch.int8).flatten(-2), (top / 127.0).squeeze(-1).half()


def _table(case, need, first, g):
    """Page tables of a batch whose pages were handed out in random order; sequences of a group begin with the same ones."""
    width = max(need)
    alone = [n - f for n, f in zip(need, first)]
    groups = list(zip(_ints(case["rows"]), _ints(case["shared"]))) if case["op"] == "shared" else []
    total = sum(alone) + sum(p // case["page"] for _, p in groups)
    perm = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.zeros(len(need), width, dtype=torch.int32, device="cuda")
    at = row = 0
    for n, p in groups:
        table[row:row + n, :p // case["page"]] = perm[at:at + p // case["page"]]
        at, row = at + p // case["page"], row + n
    start = torch.tensor([at] + alone[:-1], device="cuda").cumsum(0)[:, None]
    col = torch.arange(width, device="cuda")
    lo, hi = (torch.tensor(x, device="cuda")[:, None] for x in (first, need))
    mine = (col >= lo) & (col < hi)
    return torch.where(mine, perm[(start + col - lo).clamp(0, total - 1)], table).contiguous(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    st = dict(case=case)
    if case["op"] == "adjust":
        B, V, L, n = case["batch"], case["vocab"], case["hist"], case["bias"]
        word = lambda *s: (torch.rand(*s, generator=g, device="cuda") ** 3 * V).int().clamp_max(V - 1)  # noqa: E731
        x = rand(B, V) * 2.0
        x += 6.0 * (torch.rand(B, V, generator=g, device="cuda") < 40.0 / V) * rand(B, V).abs()
        st["logits"] = x.to(DT[case["dtype"]])
        st["tokens"] = word(B, L)  # frequent words come often, as they do in text
        st["n_tokens"] = (L - torch.randint(0, L // 2 + 1, (B,), generator=g, device="cuda")).int()
        st["n_prompt"] = (st["n_tokens"] // 2).int()
        r = torch.arange(B, device="cuda")
        st["repetition"] = 1.0 + 0.05 * (r % 7 + 1)
        st["frequency"] = 0.1 * (r % 3).float()
        st["presence"] = 0.25 * (r % 4).float()
        st["bias_tokens"] = st["bias"] = st["allowed"] = None
        if n:
            st["bias_tokens"] = word(B, n)
            st["bias_tokens"][:, n - n // 4:] = -1  # unused places of the shorter lists
            st["bias"] = rand(B, n) * 5.0
        if case["mask"]:  # words of 32, most of them empty, as a grammar's masks are
            bits = torch.randint(-2**31, 2**31, (B, (V + 31) // 32), generator=g, device="cuda").int()
            st["allowed"] = bits * (torch.rand(bits.shape, generator=g, device="cuda") < 0.2)
        return st
    q_len, kv, first = _lens(case)
    B, T, nh, nkv, hd, pg = len(q_len), sum(q_len), case["nh"], case["nkv"], case["hd"], case["page"]
    dt = DT[case["dtype"]]
    st["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    st["max_kv"] = max(kv)
    st["table"], total = _table(case, [max(1, -(-n // pg)) for n in kv], [p // pg for p in first], g)
    if case["op"] == "shared":
        st["k"], st["v"] = rand(total, pg, nkv, hd, dtype=dt), rand(total, pg, nkv, hd, dtype=dt)
        rows = _ints(case["rows"])
        st["cu_group"] = torch.tensor([0] + rows, device="cuda").cumsum(0).int()
        st["shared_len"] = torch.tensor(_ints(case["shared"]), dtype=torch.int32, device="cuda")
        st["max_rows"], st["max_shared"] = max(rows), max(_ints(case["shared"]))
        st["max_alone"] = max(n - p for n, p in zip(kv, first))
    else:
        for c in "kv":  # codes where keys and values would be, the scales of a head's positions side by side
            st[c], d = _blocks(rand(total, pg, nkv, hd, dtype=torch.float16))
            st[c + "s"] = d.transpose(1, 2).contiguous()
    if case["op"] == "store":
        st["qkv"] = rand(T, (nh + 2 * nkv) * hd).to(DT[case["src"]])
        ang = torch.arange(max(kv), device="cuda")[:, None].double() / 10000.0 ** (
            torch.arange(0, hd, 2, device="cuda").double() / hd)
        st["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        st["cu_q"] = torch.tensor([0] + q_len, device="cuda").cumsum(0).int()
        st["cu_read"] = torch.tensor([0] + kv, device="cuda").cumsum(0).int() if case["whole"] else st["cu_q"]
        st["read"] = sum(kv) if case["whole"] else T
        return st
    st["q"] = (rand(T, nh, hd) * 2.0).to(dt)  # scores of standard deviation 2: some keys matter, none is alone
    st["out"] = DT[case["out"]]
    return st


# ------------------------------------------------------------------ plain forms
def _rows_of(cu, rows):
    """(sequence, place in it, rows of it) of each packed row."""
    t, cu = torch.arange(rows, device="cuda"), cu.long()
    s = torch.searchsorted(cu, t, right=True) - 1
    return s, t - cu[s], (cu[1:] - cu[:-1])[s]


def _plain_store(st):
    case, x = st["case"], st["qkv"].float()
    nh, nkv, hd, pg, dt = case["nh"], case["nkv"], case["hd"], case["page"], DT[case["dtype"]]
    s, i, n = _rows_of(st["cu_q"], x.shape[0])
    p = st["kv_len"].long()[s] - n + i
    x = x.view(-1, nh + 2 * nkv, hd)
    qk = x[:, :nh + nkv].unflatten(-1, (hd // 2, 2))
    c, d = st["rope"][p, None, :, 0], st["rope"][p, None, :, 1]
    qk = torch.stack([qk[..., 0] * c - qk[..., 1] * d, qk[..., 0] * d + qk[..., 1] * c], -1).flatten(-2)
    page = st["table"].long()[s, p // pg]
    st["k"][page, p % pg], st["ks"][page, :, p % pg] = _blocks(qk[:, nh:])
    st["v"][page, p % pg], st["vs"][page, :, p % pg] = _blocks(x[:, nh + nkv:])
    s, i, n = _rows_of(st["cu_read"], st["read"])
    p = st["kv_len"].long()[s] - n + i
    page = st["table"].long()[s, p // pg]
    back = lambda c, d: (c[page, p % pg].float().unflatten(-1, (-1, 32)) * d[page, :, p % pg].float()[..., None])  # noqa: E731
    return qk[:, :nh].to(dt), back(st["k"], st["ks"]).flatten(-2).to(dt), back(st["v"], st["vs"]).flatten(-2).to(dt)


def _plain_paged8(st):
    """Sequences padded to the longest; keys and values in 32 bits."""
    case = st["case"]
    nh, nkv, hd, pg = case["nh"], case["nkv"], case["hd"], case["page"]
    j = torch.arange(st["max_kv"], device="cuda")
    page = st["table"].long()[:, j // pg]
    back = lambda c, d: (c[page, j % pg].float().unflatten(-1, (-1, 32)) * d[page, :, j % pg].float()[..., None]).flatten(-2)  # noqa: E731
    K = back(st["k"], st["ks"]).permute(0, 2, 3, 1)
    S = torch.matmul(st["q"].float().view(-1, nkv, nh // nkv, hd), K).mul_(1.0 / math.sqrt(hd))
    S.masked_fill_((j >= st["kv_len"].long()[:, None])[:, None, None], -math.inf)
    m = S.amax(-1, keepdim=True)
    P = S.sub_(m.masked_fill_(m == -math.inf, 0.0)).exp_()
    l = P.sum(-1, keepdim=True)
    O = torch.matmul(P, back(st["v"], st["vs"]).transpose(1, 2)) / l.masked_fill(l == 0, 1.0)
    return O.reshape(-1, nh, hd).to(st["out"])


def _plain_shared(st):
    """The prefix of each group by one product for all its sequences, the rest sequence by sequence, one softmax."""
    case, q = st["case"], st["q"]
    nh, nkv, hd, pg = case["nh"], case["nkv"], case["hd"], case["page"]
    grp, B = nh // nkv, q.shape[0]
    cu, P = st["cu_group"].long(), st["shared_len"].long()
    G, R = P.numel(), st["max_rows"]
    s = torch.arange(B, device="cuda")
    g = torch.searchsorted(cu, s, right=True) - 1
    at = lambda t, p: (t.long()[:, :, None].expand(-1, -1, pg) * pg + torch.arange(pg, device="cuda")).flatten(1).gather(1, p)  # noqa: E731
    j = torch.arange(st["max_shared"], device="cuda")
    rows = at(st["table"][cu[:-1]], j.expand(G, -1).clamp_max(st["table"].shape[1] * pg - 1))
    kv = lambda c, r: st[c].view(-1, nkv, hd)[r].float()  # noqa: E731
    Q = q[(cu[:-1, None] + torch.arange(R, device="cuda")).clamp_max(B - 1)].float().view(G, R, nkv, grp, hd)
    Q = Q.permute(0, 2, 1, 3, 4).reshape(G, nkv, R * grp, hd)
    A = torch.matmul(Q, kv("k", rows).permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(hd))
    A.masked_fill_((j >= P[:, None])[:, None, None], -math.inf)
    i = torch.arange(st["max_alone"], device="cuda")
    p = P[g][:, None] + i
    own_rows = at(st["table"], p.clamp_max(st["table"].shape[1] * pg - 1))
    C = torch.matmul(q.float().view(B, nkv, grp, hd), kv("k", own_rows).permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(hd))
    C.masked_fill_((p >= st["kv_len"].long()[:, None])[:, None, None], -math.inf)
    back = lambda t: t.view(G, nkv, R, grp, -1).permute(0, 2, 1, 3, 4)[g, s - cu[g]]  # noqa: E731  [B, nkv, grp, ...]
    pad = lambda t: torch.nn.functional.pad(t, (0, 0, 0, 0, 0, 0, 0, R))[(cu[:-1, None] + torch.arange(R, device="cuda"))]  # noqa: E731
    m = torch.maximum(back(A.amax(-1, keepdim=True)), C.amax(-1, keepdim=True))
    mg = pad(m).permute(0, 2, 1, 3, 4).reshape(G, nkv, R * grp, 1)
    A, C = A.sub_(mg).exp_(), C.sub_(m).exp_()
    l = back(A.sum(-1, keepdim=True)) + C.sum(-1, keepdim=True)
    O = back(torch.matmul(A, kv("v", rows).transpose(1, 2))) + torch.matmul(C, kv("v", own_rows).transpose(1, 2))
    return (O / l).reshape(B, nh, hd).to(st["out"])


def _plain_adjust(st):
    x = st["logits"].float()
    B, V = x.shape
    tok = st["tokens"].long()
    i = torch.arange(tok.shape[1], device="cuda")
    held = i < st["n_tokens"][:, None]
    seen = torch.zeros(B, V, dtype=torch.int32, device="cuda").scatter_add_(1, tok, held.int())
    count = torch.zeros_like(seen).scatter_add_(1, tok, (held & (i >= st["n_prompt"][:, None])).int())
    r = st["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count - torch.where(count > 0, st["presence"][:, None], 0.0)
    if st["bias"] is not None:
        used = st["bias_tokens"] >= 0
        add = torch.zeros(B, V, dtype=torch.float64, device="cuda")
        add.scatter_add_(1, st["bias_tokens"].long().clamp_min(0), torch.where(used, st["bias"], 0.0).double())
        x = x + add.float()
    if st["allowed"] is not None:
        w = torch.arange(V, device="cuda")
        x = torch.where((st["allowed"][:, w // 32] >> (w % 32)) & 1 > 0, x, -math.inf)
    return x.to(st["logits"].dtype)


# ------------------------------------------------------------------ the framework's calls
def _own(st):
    from asmllm_b200 import ops

    case = st["case"]
    if case["op"] == "adjust":
        return ops.rows_adjust(st["logits"], tokens=st["tokens"], n_tokens=st["n_tokens"], n_prompt=st["n_prompt"],
                               repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
                               bias_tokens=st["bias_tokens"], bias=st["bias"], allowed=st["allowed"])
    if case["op"] == "store":
        q = ops.rope_append_q8(st["qkv"], st["rope"], st["kv_len"], st["table"], st["k"], st["v"], st["ks"], st["vs"],
                               case["nh"], cu_q=st["cu_q"] if case["lens"] else None, q_dtype=DT[case["dtype"]])
        k, v = ops.cache_read_q8(st["k"], st["v"], st["ks"], st["vs"], st["table"], st["kv_len"], st["cu_read"],
                                 st["read"], dtype=DT[case["dtype"]])
        return q, k, v
    if case["op"] == "paged8":
        return ops.attention_paged_q8(st["q"], st["k"], st["v"], st["ks"], st["vs"], st["table"], st["kv_len"],
                                      out_dtype=st["out"])
    return ops.attention_shared(st["q"], st["k"], st["v"], st["table"], st["kv_len"], st["cu_group"],
                                st["shared_len"], out_dtype=st["out"])


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "paged8": _plain_paged8, "shared": _plain_shared,
            "adjust": _plain_adjust}[state["case"]["op"]](state)


# ------------------------------------------------------------------ work and 64-bit values
def work(case):
    if case["op"] == "adjust":
        B, n = case["batch"], case["batch"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "bf16" else 8) + B * (case["hist"] * 3 + case["bias"] * 8 + 20)
                + (n // 8 if case["mask"] else 0), "flops": 4 * n}
    q_len, kv, first = _lens(case)
    nh, nkv, hd, T = case["nh"], case["nkv"], case["hd"], sum(q_len)
    row8 = 2 * nkv * (hd + hd // 16)  # a position's codes and scales, keys and values
    if case["op"] == "store":
        n, back = (nh + 2 * nkv) * hd, sum(kv) if case["whole"] else T
        return {"bytes": T * (n * (4 if case["src"] == "fp32" else 2) + nh * hd * 2 + row8 + hd * 4)
                + back * (row8 + 4 * nkv * hd), "flops": 3 * T * (nh + nkv) * hd + 4 * T * nkv * hd + 2 * back * nkv * hd}
    io = T * nh * hd * (2 + (4 if case["out"] == "fp32" else 2))
    if case["op"] == "paged8":
        return {"bytes": io + sum(kv) * row8, "flops": 4 * sum(kv) * nh * hd}
    held = sum(_ints(case["shared"])) + sum(kv) - sum(first)
    return {"bytes": io + held * nkv * hd * 4, "flops": 4 * sum(kv) * nh * hd}


def _exact_adjust(case, st):
    y = st["logits"].double()
    for b in range(case["batch"]):
        n, m = int(st["n_tokens"][b]), int(st["n_prompt"][b])
        for w, tok in ((True, st["tokens"][b, :n]), (False, st["tokens"][b, m:n])):
            word, count = tok.long().unique(return_counts=True)
            if w:
                v, r = y[b, word], st["repetition"][b].double()
                y[b, word] = torch.where(v > 0, v / r, v * r)
            else:
                y[b, word] -= st["frequency"][b].double() * count + st["presence"][b].double()
        if st["bias"] is not None:
            use = st["bias_tokens"][b] >= 0
            y[b].index_put_((st["bias_tokens"][b][use].long(),), st["bias"][b][use].double(), accumulate=True)
        if st["allowed"] is not None:
            bit = (st["allowed"][b][:, None] >> torch.arange(32, device="cuda")) & 1
            y[b][bit.flatten()[:case["vocab"]] == 0] = -math.inf
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "adjust":
        return _exact_adjust(case, st)
    q_len, kv, _ = _lens(case)
    nh, nkv, hd, pg = case["nh"], case["nkv"], case["hd"], case["page"]
    pages = lambda s, n: st["table"][s].long()[:max(1, -(-n // pg))]  # noqa: E731

    def held(c, s, n):
        """Keys or values of the first n positions of sequence s in 64 bits."""
        x = st[c][pages(s, n)].double().flatten(0, 1)[:n]
        if c + "s" not in st:
            return x
        d = st[c + "s"][pages(s, n)].double().transpose(1, 2).flatten(0, 1)[:n]
        return x * d.repeat_interleave(32, -1)

    at, outs = 0, []
    if case["op"] == "store":
        back = {"k": [], "v": []}
        x = st["qkv"].double().view(-1, nh + 2 * nkv, hd)
        for s, (n, m) in enumerate(zip(q_len, kv)):
            rows, p = x[at:at + n], torch.arange(m - n, m, device="cuda")
            z = torch.view_as_complex(rows[:, :nh + nkv].unflatten(-1, (hd // 2, 2)).contiguous())
            z = torch.view_as_real(z * torch.view_as_complex(st["rope"].double().contiguous())[p][:, None]).flatten(-2)
            outs.append(z[:, :nh])
            for c, new in (("k", z[:, nh:]), ("v", rows[:, nh + nkv:])):
                b = new.unflatten(-1, (-1, 32))
                a = b.abs().amax(-1, keepdim=True)
                new = (torch.round(b * 127.0 / a.clamp_min(1e-300)) * (a / 127.0).half().double()).flatten(-2)
                back[c].append(torch.cat([held(c, s, m)[:m - n], new]) if case["whole"] else new)
            at += n
        return torch.cat(outs), torch.cat(back["k"]), torch.cat(back["v"])
    for s, m in enumerate(kv):
        q, k, v = st["q"][s].double().view(nkv, nh // nkv, hd), held("k", s, m), held("v", s, m)
        a = torch.einsum("jgd,pjd->jgp", q, k) * hd ** -0.5
        outs.append(torch.einsum("jgp,pjd->jgd", torch.softmax(a, -1), v).reshape(nh, hd))
    return torch.stack(outs)
