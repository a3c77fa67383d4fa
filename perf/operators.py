"""The attention operators as cases that can be timed and compared.

A case is one pass of one operator over a batch of sequences with a paged cache: ``append`` norms and rotates
the batch's query and key heads and writes keys and values into the cache's pages, ``attend`` is the attention
of the batch's tokens over the cache. Every token sees the positions of its own sequence up to its own. Where
sequences share a prefix their page tables start with the same pages.

The cache lies as the library keeps it: keys [page][kv head][slot][D], values [page][kv head][D][slot]. A case's
sequence lengths follow from the case; a seed makes the values and deals the pages."""
import math

import numpy as np
import torch

own = False

HEADS = {  # query heads, kv heads, width of a head
    "small": (14, 2, 64),      # generic: seven query heads on a kv head
    "mha": (16, 16, 128),      # generic: as many kv heads as query heads
    "q30b": (32, 4, 128),      # Qwen3-30B-A3B
    "q235b": (64, 4, 128),     # Qwen3-235B-A22B
}
TYPES = {"f16": torch.float16, "f32": torch.float32}
BASE, EPS = 1e6, 1e-6


def listed():
    return [
        # one sequence's next token: launch and latency
        {"name": "append_t1", "op": "append", "heads": "q30b", "cache": "f16", "page": 64, "seqs": 1, "q": 1, "past": 4320, "prefix": 0, "ragged": False},
        # a serving batch's next tokens, each at its own position
        {"name": "append_t64", "op": "append", "heads": "q235b", "cache": "f16", "page": 64, "seqs": 64, "q": 1, "past": 4095, "prefix": 0, "ragged": True},
        # a piece of a long document, far into the context
        {"name": "append_t2047_far", "op": "append", "heads": "q235b", "cache": "f16", "page": 128, "seqs": 1, "q": 2047, "past": 129000, "prefix": 0, "ragged": False},
        # a few odd-sized prompts on the fp32 cache of the reference's kind
        {"name": "append_f32_prompts", "op": "append", "heads": "small", "cache": "f32", "page": 16, "seqs": 3, "q": 201, "past": 0, "prefix": 0, "ragged": True},
        # chat: one sequence of the smaller model early in its context
        {"name": "decode_513", "op": "attend", "heads": "q30b", "cache": "f16", "page": 64, "seqs": 1, "q": 1, "past": 512, "prefix": 0, "ragged": False},
        # a serving batch of mixed lengths
        {"name": "decode_b32", "op": "attend", "heads": "q235b", "cache": "f16", "page": 64, "seqs": 32, "q": 1, "past": 8190, "prefix": 0, "ragged": True},
        # one long context
        {"name": "decode_long", "op": "attend", "heads": "q235b", "cache": "f16", "page": 128, "seqs": 1, "q": 1, "past": 131070, "prefix": 0, "ragged": False},
        # drafted tokens checked in one pass
        {"name": "draft_b8", "op": "attend", "heads": "q235b", "cache": "f16", "page": 64, "seqs": 8, "q": 5, "past": 4003, "prefix": 0, "ragged": True},
        # a prompt from its start
        {"name": "prompt_2047", "op": "attend", "heads": "q235b", "cache": "f16", "page": 64, "seqs": 1, "q": 2047, "past": 0, "prefix": 0, "ragged": False},
        # a piece of a long prompt
        {"name": "chunk_509", "op": "attend", "heads": "q30b", "cache": "f16", "page": 32, "seqs": 1, "q": 509, "past": 16000, "prefix": 0, "ragged": False},
        # many answers to one long document
        {"name": "shared_b64", "op": "attend", "heads": "q235b", "cache": "f16", "page": 64, "seqs": 64, "q": 1, "past": 8703, "prefix": 8192, "ragged": True},
        # odd-sized prompts on the fp32 cache
        {"name": "prompts_f32", "op": "attend", "heads": "small", "cache": "f32", "page": 16, "seqs": 3, "q": 701, "past": 0, "prefix": 0, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = {"op": rng.choice(["append", "attend", "attend"]), "heads": rng.choice(list(HEADS)),
            "cache": rng.choice(["f16", "f16", "f16", "f32"]), "page": rng.choice([16, 32, 64, 128, 256])}
    kind = rng.choice(["decode", "decode", "draft", "prompt", "chunk", "shared"])
    page = case["page"]
    prefix = 0
    if kind == "decode":
        seqs, q, past = _log_int(rng, 1, 64), 1, _log_int(rng, 1, 131070)
    elif kind == "draft":
        seqs, q, past = _log_int(rng, 1, 32), rng.randint(2, 8), _log_int(rng, 16, 16000)
    elif kind == "prompt":
        seqs, q, past = _log_int(rng, 1, 8), _log_int(rng, 9, 2047), 0
    elif kind == "chunk":
        seqs, q, past = _log_int(rng, 1, 2), _log_int(rng, 9, 1021), _log_int(rng, 33, 16000)
    else:
        seqs, q, past = _log_int(rng, 4, 64), rng.choice([1, 1, 1, 3]), _log_int(rng, 1023, 16000)
        prefix = int(past * rng.uniform(0.5, 0.97)) // page * page
    case.update(seqs=seqs, q=q, past=past, prefix=prefix, ragged=rng.random() < 0.7)
    while _too_big(case):          # no dearer than the largest listed case
        if case["seqs"] > 1:
            case["seqs"] = case["seqs"] * 3 // 4
        else:
            case["past"] = case["past"] * 3 // 4
            case["q"] = min(case["q"], max(1, case["q"] * 7 // 8))
        case["prefix"] = min(case["prefix"], case["past"] // page * page)
    return case


def _too_big(case):
    Hq, Hkv, D = HEADS[case["heads"]]
    w = work(dict(case, op="attend"))
    flops = w["flops"] * (4 if case["cache"] == "f32" else 1)
    lens = _lens(case)
    gathered = len(lens) * max(q + p for q, p in lens) * Hkv * D
    scores = len(lens) * max(q for q, _ in lens) * max(q + p for q, p in lens) * Hq
    return flops > 1.35e11 or w["bytes"] > 2.7e8 or gathered > 2.85e8 or scores > 2.8e8


def _lens(case):
    """(new tokens, earlier tokens) of each sequence; ragged ones are spread by steps of the golden section."""
    out = []
    for i in range(case["seqs"]):
        f = 1.0 - (i * 0.6180339887498949) % 1.0 if case["ragged"] else 1.0
        q = case["q"] if case["q"] <= 8 else max(1, int(case["q"] * f))
        out.append((q, case["prefix"] + int((case["past"] - case["prefix"]) * f)))
    return out


# ---- what a program has in hand ----

def _inputs(case, seed):
    """Page tables, pools and the batch's rows. Pools hold a page more than the batch's own."""
    Hq, Hkv, D = HEADS[case["heads"]]
    page, dtype = case["page"], TYPES[case["cache"]]
    g = torch.Generator("cuda").manual_seed(int(seed))
    lens = _lens(case)
    shared = case["prefix"] // page
    need = [-(-(q + p) // page) for q, p in lens]
    n_page = shared + sum(n - shared for n in need) + 1
    deal = np.random.RandomState(int(seed) % (1 << 31)).permutation(n_page)
    table = np.zeros((len(lens), max(need)), np.int32)
    at = shared
    for i, n in enumerate(need):
        table[i, :shared] = deal[:shared]
        table[i, shared:n] = deal[at:at + n - shared]
        at += n - shared
    T = sum(q for q, _ in lens)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    st = {"table": table, "lens": lens, "n_page": n_page,
          "kpool": normal(n_page, Hkv, page, D).to(dtype), "vpool": normal(n_page, Hkv, D, page).to(dtype)}
    if case["op"] == "append":
        st.update(q=normal(T, Hq * D), k=normal(T, Hkv * D) * 3, v=normal(T, Hkv * D), qw=1 + 0.3 * normal(D), kw=1 + 0.3 * normal(D))
    else:
        st["q"] = normal(T, Hq * D) * 2        # normed heads times their weights: scores of a few units
    return st


def _index(lens):
    """Per token its sequence and position; per (sequence, new token) the token's row, padded with row 0."""
    seq = np.concatenate([np.full(q, i) for i, (q, _) in enumerate(lens)])
    pos = np.concatenate([p + np.arange(q) for q, p in lens])
    row = np.zeros((len(lens), max(q for q, _ in lens)), np.int64)
    limit = np.zeros_like(row)
    at = 0
    for i, (q, p) in enumerate(lens):
        row[i, :q], limit[i, :q] = at + np.arange(q), p + 1 + np.arange(q)
        at += q
    return seq, pos, row, limit


def prepare(case, seed):
    Hq, Hkv, D = HEADS[case["heads"]]
    st = _inputs(case, seed)
    st["case"] = case
    st["out"] = torch.empty_like(st["q"])
    seq, pos, row, limit = (torch.from_numpy(a).cuda() for a in _index(st["lens"]))
    tab = torch.from_numpy(st["table"].astype(np.int64)).cuda()
    st.update(pos=pos, row=row, limit=limit, tab=tab, page_of=tab[seq, pos // case["page"]], slot=pos % case["page"])
    if own:
        from large_model_amd import qmsg
        ctx = qmsg.Context(256, 16, 4, 128, n_layer=1, max_tokens=1)
        a = ctx.attn_create(Hq, Hkv, D, type_=qmsg.QMSG_T_F16 if case["cache"] == "f16" else qmsg.QMSG_T_F32,
                            page=case["page"], n_page=st["n_page"], n_layer=1, rope_base=BASE, qk_norm=True,
                            max_seq=len(st["lens"]), max_tokens=st["q"].shape[0], max_pages=st["table"].shape[1],
                            d_k=st["kpool"].data_ptr(), d_v=st["vpool"].data_ptr())
        if case["op"] == "append":
            ctx.attn_norms(a, 0, st["qw"].cpu().numpy(), st["kw"].cpu().numpy())
        ctx.attn_batch(a, [q for q, _ in st["lens"]], [q + p for q, p in st["lens"]], st["table"])
        st.update(ctx=ctx, attn=a)
    torch.cuda.synchronize()           # the library works on its context's own stream
    return st


# ---- one pass ----

def run(st):
    case = st["case"]
    if case["op"] == "append":
        if own:
            st["ctx"].attn_append_device(st["attn"], 0, st["out"].data_ptr(), st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), EPS)
        else:
            _append(st)
        return {"q": st["out"], "k": st["kpool"], "v": st["vpool"]}
    if own:
        st["ctx"].attn_device(st["attn"], 0, st["q"].data_ptr(), st["out"].data_ptr())
        return st["out"]
    return _attend(st)


def _heads(x, w, pos, D):
    """Normed and rotated heads of x [T][H * D]."""
    x = x.reshape(x.shape[0], -1, D)
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
    angle = pos.double()[:, None] * BASE ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(st):
    Hq, Hkv, D = HEADS[st["case"]["heads"]]
    st["out"].copy_(_heads(st["q"], st["qw"], st["pos"], D).reshape(-1, Hq * D))
    st["kpool"][st["page_of"], :, st["slot"]] = _heads(st["k"], st["kw"], st["pos"], D).to(st["kpool"].dtype)
    st["vpool"][st["page_of"], :, :, st["slot"]] = st["v"].reshape(-1, Hkv, D).to(st["vpool"].dtype)


def _attend(st):
    Hq, Hkv, D = HEADS[st["case"]["heads"]]
    G, (B, Q) = Hq // Hkv, st["row"].shape
    k = st["kpool"][st["tab"]].float().transpose(1, 2).reshape(B, Hkv, -1, D)
    v = st["vpool"][st["tab"]].float().permute(0, 2, 1, 4, 3).reshape(B, Hkv, -1, D)
    q = st["q"].reshape(-1, Hkv, G, D)[st["row"]].transpose(1, 2).reshape(B, Hkv, Q * G, D)
    s = (q @ k.transpose(-1, -2).contiguous()) * D ** -0.5
    seen = torch.arange(k.shape[2], device="cuda") < st["limit"].repeat_interleave(G, 1)[:, None, :, None]
    s = s.masked_fill_(~seen, -torch.inf)
    e = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()      # padded tokens see nothing
    o = (e @ v) / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.reshape(B, Hkv, Q, G, D).transpose(1, 2).reshape(B, Q, Hq * D)
    return o[st["limit"] > 0]


# ---- what a pass cannot do without ----

def work(case):
    Hq, Hkv, D = HEADS[case["heads"]]
    e = 2 if case["cache"] == "f16" else 4
    lens = _lens(case)
    T = sum(q for q, _ in lens)
    if case["op"] == "append":
        return {"bytes": 4 * T * D * (2 * Hq + 2 * Hkv) + 2 * e * T * D * Hkv, "flops": 8 * T * D * (Hq + Hkv)}
    keys = case["prefix"] + sum(q + p - case["prefix"] for q, p in lens)
    seen = sum(q * p + q * (q + 1) // 2 for q, p in lens)
    return {"bytes": 2 * e * keys * D * Hkv + 8 * T * D * Hq, "flops": 4 * D * Hq * seen}


# ---- the same in float64 ----

def _exact_heads(x, w, pos, D):
    h = D // 2
    x = x.double().reshape(len(x), -1, D)
    y = x / ((x * x).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
    turn = torch.exp(-math.log(BASE) / h * torch.arange(h, device="cuda", dtype=torch.float64))
    z = torch.polar(torch.ones(len(pos), h, device="cuda", dtype=torch.float64), torch.outer(pos.double(), turn))
    r = torch.complex(y[..., :h], y[..., h:]) * z[:, None]
    return torch.cat([r.real, r.imag], -1)


def exact(case, seed):
    Hq, Hkv, D = HEADS[case["heads"]]
    G, page = Hq // Hkv, case["page"]
    st = _inputs(case, seed)
    if case["op"] == "append":
        seq, pos, _, _ = _index(st["lens"])
        kpool, vpool = st["kpool"].double(), st["vpool"].double()
        pt = torch.from_numpy(pos).cuda()
        k, v = _exact_heads(st["k"], st["kw"], pt, D), st["v"].double().reshape(-1, Hkv, D)
        at = torch.from_numpy(st["table"][seq, pos // page].astype(np.int64) * page + pos % page).cuda()
        kpool[at // page, :, at % page] = k
        vpool[at // page, :, :, at % page] = v
        return {"q": _exact_heads(st["q"], st["qw"], pt, D).reshape(-1, Hq * D), "k": kpool, "v": vpool}
    out, at = [], 0
    for i, (q, p) in enumerate(st["lens"]):
        pages = torch.from_numpy(st["table"][i, :-(-(q + p) // page)].astype(np.int64)).cuda()
        K = st["kpool"][pages].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :q + p]
        V = st["vpool"][pages].double().permute(1, 2, 0, 3).reshape(Hkv, D, -1)[:, :, :q + p]
        x = st["q"][at:at + q].double().reshape(q, Hkv, G, D)
        at += q
        step = max(1, int(2e8 // (Hq * (q + p))))
        for a in range(0, q, step):
            rows = x[a:a + step].transpose(0, 1)                      # kv head, token, group, D
            n = rows.shape[1]
            s = torch.matmul(rows.reshape(Hkv, n * G, D), K.transpose(1, 2).contiguous()) / math.sqrt(D)
            s = s.reshape(Hkv, n, G, q + p)
            hidden = torch.arange(q + p, device="cuda")[None, :] > (p + a + torch.arange(n, device="cuda"))[:, None]
            w = torch.softmax(s.masked_fill(hidden[None, :, None], -math.inf), -1).reshape(Hkv, n * G, q + p)
            o = torch.matmul(w, V.transpose(1, 2).contiguous())
            out.append(o.reshape(Hkv, n, G, D).transpose(0, 1).reshape(n, Hq * D))
    return torch.cat(out)
