"""The operators of serving and scoring over a cache held in 8 bits, as cases that can be timed and compared.

A program that keeps its own projections appends the new keys and values of its sequences to a paged cache
(e4m3 values, one power-of-two scale for each page and kv head), rotating queries and keys by their positions
on the way, and attends over that cache; from the logits it takes the log probabilities of the tokens it
scores, with each row's entropy and its most probable alternatives.  Heads, vocabulary, prefixes and block
sizes are the 1.5B configuration's and the benchmark's (12 query heads on 2 kv heads of 128, prefixes of 512
to 8192 rows, blocks of 32 and sub-blocks of 8, 16 sequences with prefixes in [128, 1024], continuations of
64 tokens, a context window of 32768), and generic ones beside them.

Layout of one layer's pages: keys [pages, kv heads, page, 128] and values [pages, kv heads, 128, page], both
e4m3; scales [pages, kv heads] fp32 for each.  Position p of a sequence is slot p % page of the page that its
row of the page table names at p // page.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

DEV = "cuda"
HD = 128
VOCAB = 151936
THETA = 1e6
LAYERS, LAYER = 2, 1  # the caches hold two layers; the calls take the second
TD = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
FP8 = torch.float8_e4m3fn

# a case's fields: `nq` / `nkv` heads; `page` tokens a page; `nseq` sequences, whose cached lengths before the
# call come from [lo, hi] with `lens`; `rows` new rows of each (up to that many where `ragged`); `rp` the row
# of a block that is live already at which the new rows start; `mask` 0 none, else block-causal in blocks of
# that many positions (1: causal); log probabilities: `rows` x `vocab` logits in `dtype`, `top` alternatives


def listed():
    return [
        # one sequence's next token, once a layer: latency
        dict(name="append_1x1", kind="append", nq=12, nkv=2, page=32, nseq=1, lo=2079, hi=2079, lens=1, rows=1, rp=0,
             ragged=False, dtype="bfloat16"),
        # a sub-block refined again in blocks that the pages hold already, after prompts that end inside a page
        dict(name="append_16x8", kind="append", nq=12, nkv=2, page=32, nseq=16, lo=128, hi=1024, lens=3, rows=8, rp=8,
             ragged=False, dtype="float16"),
        # prompts of many lengths appended in one call
        dict(name="append_ragged", kind="append", nq=12, nkv=2, page=64, nseq=24, lo=0, hi=700, lens=5, rows=509, rp=0,
             ragged=True, dtype="bfloat16"),
        # the longest prompt
        dict(name="append_8192", kind="append", nq=12, nkv=2, page=32, nseq=1, lo=0, hi=0, lens=1, rows=8192, rp=0,
             ragged=False, dtype="bfloat16"),
        # one sequence's next token over an ordinary prompt: latency
        dict(name="attn_1x1_p2080", kind="attn", nq=12, nkv=2, page=32, nseq=1, lo=2079, hi=2079, lens=1, rows=1,
             mask=0, ragged=False, dtype="bfloat16"),
        # many sequences' blocks refined together
        dict(name="attn_16x32", kind="attn", nq=12, nkv=2, page=32, nseq=16, lo=128, hi=1024, lens=3, rows=32,
             mask=0, ragged=False, dtype="float16"),
        # a block after a prompt that fills the context window
        dict(name="attn_1x32_p32736", kind="attn", nq=12, nkv=2, page=32, nseq=1, lo=32736, hi=32736, lens=1, rows=32,
             mask=0, ragged=False, dtype="bfloat16"),
        # many sequences' next tokens over long prompts: the cache's bytes
        dict(name="attn_64x1_p8192", kind="attn", nq=12, nkv=2, page=64, nseq=64, lo=1024, hi=8191, lens=7, rows=1,
             mask=1, ragged=False, dtype="bfloat16"),
        # the last part of a long prompt, block-causal
        dict(name="attn_2048_p8192", kind="attn", nq=12, nkv=2, page=32, nseq=1, lo=6144, hi=6144, lens=1, rows=2048,
             mask=32, ragged=False, dtype="bfloat16"),
        # one generated token with the usual number of alternatives, from 16-bit logits of an odd vocabulary
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=151643, top=20, dtype="bfloat16"),
        # scoring a continuation of 64 tokens
        dict(name="logprobs_64", kind="logprobs", rows=64, vocab=VOCAB, top=5, dtype="float32"),
        # scoring many continuations
        dict(name="logprobs_1024", kind="logprobs", rows=1024, vocab=VOCAB, top=20, dtype="float32"),
    ]


def _log_size(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng: random.Random):
    kind = rng.choice(("append", "attn", "attn", "logprobs"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    if kind == "logprobs":
        return dict(kind=kind, rows=_log_size(rng, 1, 600), vocab=_log_size(rng, 1000, VOCAB),
                    top=rng.choice((0, 1, 5, 20, 32)), dtype=rng.choice(("float32", "float32", dtype)))
    nq, nkv = rng.choice(((12, 2), (12, 2), (4, 2), (8, 8), (16, 1)))
    nseq = _log_size(rng, 1, 64)
    rows = rng.choice((1, 8, 32, _log_size(rng, 1, max(1, 4096 // nseq))))
    lo = _log_size(rng, 1, 8192 // nseq + 64)
    c = dict(kind=kind, nq=nq, nkv=nkv, page=rng.choice((16, 32, 32, 64, 128)), nseq=nseq, lo=lo,
             hi=lo + _log_size(rng, 1, 40000 // nseq), lens=rng.randrange(1 << 20), rows=rows,
             ragged=rng.random() < 0.3, dtype=dtype)
    if kind == "append":
        return dict(c, rp=rng.choice((0, 0, 8)) if rows <= 24 else 0)
    return dict(c, mask=rng.choice((0, 1, 32)))


# ---- what a case's sizes come to ---------------------------------------------------------------------------


def _plan(case):
    """Per sequence: first cached position of the new rows, live rows before the call, new rows."""
    rng = random.Random(case["lens"])
    pre = [rng.randint(case["lo"], case["hi"]) for _ in range(case["nseq"])]
    n = [rng.randint(0, case["rows"]) if case["ragged"] else case["rows"] for _ in pre]
    if case["ragged"]:
        n[-1] = case["rows"]
    if case["kind"] == "append":
        start = [p + case["rp"] for p in pre]
        live = [p + 32 if case["rp"] else p for p in pre]
        return start, live, n
    return pre, [p + k for p, k in zip(pre, n)], n


def _pairs(case):
    """(query row, key) pairs that the attention takes."""
    pre, total, n = _plan(case)
    b, pairs = case["mask"], 0
    for p, t, k in zip(pre, total, n):
        pairs += k * t if not b else sum(min(t, ((p + i) // b + 1) * b) for i in range(k))
    return pairs


def work(case):
    if case["kind"] == "logprobs":
        n, size = case["rows"] * case["vocab"], 4 if case["dtype"] == "float32" else 2
        return dict(bytes=n * size + case["rows"] * (12 + 8 * case["top"]), flops=5 * n)
    nq, nkv, page = case["nq"], case["nkv"], case["page"]
    a, total, n = _plan(case)
    rows = sum(n)
    if case["kind"] == "append":
        # q, k and v read, q written in 16 bits; k and v written in 8, with the scales of their pages read and written
        pages = sum((s + k - 1) // page - s // page + 1 for s, k in zip(a, n) if k)
        return dict(bytes=rows * HD * (4 * nq + 6 * nkv) + 16 * nkv * pages, flops=rows * HD * (3 * nq + 5 * nkv))
    seen = sum(t for t, k in zip(total, n) if k)
    return dict(bytes=seen * nkv * 2 * HD + 8 * nkv * (seen // page + 1) + 4 * rows * nq * HD, flops=4 * HD * nq * _pairs(case))


# ---- inputs ------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages_of(x, live, fill):
    """Rows x [pages, kv heads, page, 128] as e4m3 with a power-of-two scale for each page and head; slots that
    are not live hold what earlier owners of the page left there (here: the byte `fill`)."""
    amax = x.abs().amax(dim=(2, 3)).clamp_min(1e-20)
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448)))
    q = (x / scale[:, :, None, None]).to(FP8).view(torch.uint8)
    return torch.where(live[:, None, :, None], q, torch.full_like(q, fill)).view(FP8), scale


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # logits as the head gives them, rounded to the model's 16 bits (so equal ones are common); a few tokens
        # that a program has ruled out, and rows of padding without a token
        logits = _normal(g, (1, rows, vocab), 2.5).to(torch.bfloat16).to(TD[case["dtype"]])
        ids = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
        banned = torch.randint(0, vocab, (max(1, vocab // 1000),), generator=g, device=DEV)
        logits[:, :, banned] = -math.inf
        logits.scatter_(2, ids.long()[None, :, None], 3.0)
        if rows > 8:
            ids[5::9] = -1
        return dict(case, logits=logits, ids=ids[None])
    nq, nkv, page, nseq = case["nq"], case["nkv"], case["page"], case["nseq"]
    td = TD[case["dtype"]]
    a, total, n = _plan(case)
    rows = sum(n) + (3 if case["ragged"] else 0)  # ragged batches come padded
    # the projections of a step: one fused [q | k | v] row each, queries and keys before their rotation
    qkv = _normal(g, (rows, (nq + 2 * nkv) * HD))
    qkv *= torch.exp(_normal(g, (rows, 1), 0.5))
    need = [-(-(max(t, s + k) if case["kind"] == "append" else t) // page) for s, t, k in zip(a, total, n)]
    width = max(need) + 1
    pool = sum(need) + 2
    perm = torch.randperm(pool, generator=g, device=DEV).to(torch.int32).tolist()
    table = torch.full((nseq, width), -1, dtype=torch.int32)
    live_slots = torch.zeros((pool, page), dtype=torch.bool)
    at = 0
    for b in range(nseq):
        ids = torch.tensor(perm[at:at + need[b]], dtype=torch.int32)
        at += need[b]
        table[b, :need[b]] = ids
        slots = torch.arange(need[b] * page).view(need[b], page) < total[b]
        live_slots[ids.long()] = slots
    live_slots = live_slots.to(DEV)
    k8, ks = _pages_of(_normal(g, (pool, nkv, page, HD)), live_slots, 0x7F)
    v8, vs = _pages_of(_normal(g, (pool, nkv, page, HD), 0.7), live_slots, 0x7F)
    k = torch.empty((LAYERS, pool, nkv, page, HD), dtype=FP8, device=DEV)
    v = torch.empty((LAYERS, pool, nkv, HD, page), dtype=FP8, device=DEV)
    k.view(torch.uint8)[:] = k8.view(torch.uint8)
    v.view(torch.uint8)[:] = v8.view(torch.uint8).transpose(2, 3)
    scales = [s[None].repeat(LAYERS, 1, 1).contiguous() for s in (ks, vs)]
    starts = [0]
    for c in n:
        starts.append(starts[-1] + c)
    s = dict(case, k_pages=k, v_pages=v, k_scale=scales[0], v_scale=scales[1], table=table.to(DEV),
             row_start=_i32(starts) if case["ragged"] else None, max_rows=max(n),
             q_out=torch.zeros((rows, nq, HD), dtype=td, device=DEV))
    if case["kind"] == "append":
        qkv = qkv.to(td)
        heads = qkv.view(rows, nq + 2 * nkv, HD)
        return dict(s, q=heads[:, :nq], knew=heads[:, nq:nq + nkv], vnew=heads[:, nq + nkv:], start=_i32(a),
                    live=_i32(total))
    return dict(s, q=qkv[:, :nq * HD].reshape(rows, nq, HD).to(td), kv_len=_i32(total))


# ---- the framework's calls ---------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _vm(dtype, nq, nkv):
    """The function table a program keeps: a small model with these heads."""
    import __graft_entry__

    __graft_entry__.load_package()
    from fast_dllm_relax_amd.config import FastDLLMConfig
    from fast_dllm_relax_amd.params import TORCH_DTYPES, param_names, param_shapes
    from fast_dllm_relax_amd.vm import HipVM

    cfg = FastDLLMConfig(vocab_size=256, hidden_size=128, intermediate_size=128, num_hidden_layers=LAYERS,
                         num_attention_heads=nq, num_key_value_heads=nkv, head_dim=HD, rope_theta=THETA)
    shapes = param_shapes(cfg)
    return HipVM(cfg, [torch.zeros(shapes[n], dtype=TORCH_DTYPES[dtype], device=DEV) for n in param_names(cfg)], dtype=dtype)


def _cache(s):
    """The cache object that a program makes once over its pages."""
    if "cache" not in s:
        from fast_dllm_relax_amd.paged import PagedKVCache

        s["cache"] = PagedKVCache(k=s["k_pages"], v=s["v_pages"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s["cache"]


def _run_own(s):
    if s["kind"] == "logprobs":
        return _vm("bfloat16", 12, 2).token_logprobs(s["logits"], s["ids"], top_n=s["top"])
    vm = _vm(s["dtype"], s["nq"], s["nkv"])
    if s["kind"] == "append":
        q = vm.paged_kv_append(s["knew"], s["vnew"], _cache(s), LAYER, s["table"], s["start"], live=s["live"], q=s["q"],
                               q_out=s["q_out"], row_start=s["row_start"], max_rows=s["max_rows"])
        return q, s["k_pages"][LAYER], s["v_pages"][LAYER], s["k_scale"][LAYER], s["v_scale"][LAYER]
    return vm.paged_attn(s["q"], _cache(s), LAYER, s["table"], s["kv_len"], mask_block=s["mask"], out=s["q_out"],
                         row_start=s["row_start"], max_rows=s["max_rows"])


# ---- the plain forms ---------------------------------------------------------------------------------------


def _spread(s, rows):
    """Index of each sequence's row i among the call's rows, [nseq, max_rows], and which of them there are."""
    i = torch.arange(s["max_rows"], device=DEV)[None]
    if s["row_start"] is None:
        at = torch.arange(s["nseq"], device=DEV)[:, None] * s["max_rows"] + i
        return at, torch.ones_like(at, dtype=torch.bool)
    first, last = s["row_start"][:-1, None], s["row_start"][1:, None]
    return (first + i).clamp_max(rows - 1), first + i < last


def _plain_rotate(x, pos):
    """x [n, heads, 128] at positions pos [n], in 64 bits (far positions' angles need them)."""
    turn = pos.double()[:, None] * torch.pow(torch.tensor(THETA, dtype=torch.float64, device=DEV),
                                             -torch.arange(HD // 2, dtype=torch.float64, device=DEV) / (HD // 2))
    c, n = torch.cos(turn)[:, None], torch.sin(turn)[:, None]
    x1, x2 = x[..., :HD // 2].double(), x[..., HD // 2:].double()
    return torch.cat((x1 * c - x2 * n, x2 * c + x1 * n), dim=-1)


def _pow2_scale(amax):
    """The least power of two s with amax <= 448 s (448 = 0.875 x 2^9)."""
    m, e = torch.frexp(amax.double())
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), -100)
    return torch.exp2(e.clamp(-100, 118).double())


def _plain_append_one(s, rows, pages8, scale, page_rows, seen, old):
    """New rows (64 bits) [nseq, pages, page, heads, 128] at `seen` slots into the pages of the table."""
    seen_, old_ = seen[:, :, None, :, None], old[:, :, None, :, None]
    new = rows.permute(0, 1, 3, 2, 4)
    s_old = scale[page_rows].double()
    s_new = _pow2_scale(torch.where(seen_, new.abs(), 0).amax(dim=(3, 4)))
    has_old = old.any(dim=2)[:, :, None]
    s_all = torch.where(has_old, torch.maximum(s_old, s_new), s_new)
    held = pages8[page_rows]
    moved = (held.double() * (s_old / s_all)[..., None, None]).float().to(FP8)
    fresh = (new / s_all[..., None, None]).float().to(FP8)
    out = torch.where(seen_, fresh.view(torch.uint8),
                      torch.where(old_ & (s_all > s_old)[..., None, None], moved.view(torch.uint8), held.view(torch.uint8)))
    return out, s_all.float()


def _run_append(s):
    rows, page, nseq = s["q"].shape[0], s["page"], s["nseq"]
    at, there = _spread(s, rows)
    pos = s["start"][:, None] + torch.arange(s["max_rows"], device=DEV)[None]
    flat, src, p = there.reshape(-1), at.reshape(-1), pos.reshape(-1)
    src, p = src[flat], p[flat]
    q_out = s["q_out"]
    q_out[src] = _plain_rotate(s["q"][src], p).to(q_out.dtype)
    # the new rows laid out by sequence, page and slot
    width = s["table"].shape[1]
    seq = torch.arange(nseq, device=DEV)[:, None].expand_as(at).reshape(-1)[flat]
    slot = seq * (width * page) + p
    seen = torch.zeros(nseq * width * page, dtype=torch.bool, device=DEV)
    seen[slot] = True
    seen = seen.view(nseq, width, page)
    where = torch.arange(width * page, device=DEV).view(1, width, page)
    old = (where < s["live"][:, None, None]) & ~seen
    hit = seen.any(dim=2)
    which = s["table"][hit].long()
    for x, pages, scale in ((_plain_rotate(s["knew"][src], p), s["k_pages"][LAYER], s["k_scale"][LAYER]),
                            (s["vnew"][src].double(), s["v_pages"][LAYER].transpose(2, 3), s["v_scale"][LAYER])):
        new = torch.zeros((nseq * width * page, s["nkv"], HD), dtype=torch.float64, device=DEV)
        new[slot] = x
        new = new.view(nseq, width, page, s["nkv"], HD)[hit][:, None]
        out, sc = _plain_append_one(s, new, pages, scale, which[:, None], seen[hit][:, None], old[hit][:, None])
        pages.view(torch.uint8)[which] = out[:, 0]
        scale[which] = sc[:, 0]
    return q_out, s["k_pages"][LAYER], s["v_pages"][LAYER], s["k_scale"][LAYER], s["v_scale"][LAYER]


def _run_attn(s):
    rows, nq, nkv, page, nseq = s["q"].shape[0], s["nq"], s["nkv"], s["page"], s["nseq"]
    group, width = nq // nkv, s["table"].shape[1]
    at, there = _spread(s, rows)
    keys = torch.arange(width * page, device=DEV)
    live = keys[None] < s["kv_len"][:, None]
    ids = s["table"].clamp_min(0).long()
    k = s["k_pages"][LAYER][ids].float() * s["k_scale"][LAYER][ids][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(nseq, nkv, width * page, HD)
    v = s["v_pages"][LAYER][ids].float() * s["v_scale"][LAYER][ids][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(nseq, nkv, width * page, HD)
    k = torch.where(live[:, None, :, None], k, 0.0)
    v = torch.where(live[:, None, :, None], v, 0.0)
    q = s["q"][at].float().view(nseq, s["max_rows"], nkv, group, HD).permute(0, 2, 1, 3, 4)
    q = q.reshape(nseq, nkv, s["max_rows"] * group, HD)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(HD))
    count = there.sum(dim=1)
    pos = (s["kv_len"] - count)[:, None] + torch.arange(s["max_rows"], device=DEV)[None]
    see = live[:, None, :].expand(nseq, s["max_rows"], width * page)
    if s["mask"]:
        see = see & (keys[None, None] < ((pos // s["mask"] + 1) * s["mask"])[:, :, None])
    score = torch.where(see[:, None, :, None], score.view(nseq, nkv, s["max_rows"], group, -1), -math.inf)
    top = score.amax(dim=-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(score - top)
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(nseq, nkv, s["max_rows"] * group, -1), v).view(nseq, nkv, s["max_rows"], group, HD)
    o = o.permute(0, 2, 1, 3, 4).reshape(nseq, s["max_rows"], nq, HD)
    out = s["q_out"]
    out[at[there]] = o[there].to(out.dtype)
    return out


def _run_logprobs(s):
    x, ids, top = s["logits"].float() + 0.0, s["ids"], s["top"]  # (no -0: it equals +0)
    vocab = x.shape[-1]
    m = x.amax(dim=-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(dim=-1, keepdim=True)
    lse = torch.log(total)
    entropy = (lse - torch.where(e > 0, e * d, 0.0).sum(dim=-1, keepdim=True) / total)[..., 0]
    # a row without a token (id < 0) scores 0
    logprob = torch.gather(d, -1, ids.long().clamp_min(0)[..., None])[..., 0] - lse[..., 0]
    logprob = torch.where(ids < 0, 0.0, logprob)
    # alternatives by value, equal ones by index: one sortable key for both
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 31) - torch.arange(vocab, device=DEV)
    at = torch.topk(key, top, dim=-1).indices if top else torch.empty((*ids.shape, 0), dtype=torch.int64, device=DEV)
    return logprob, entropy, at.to(torch.int32), torch.gather(d, -1, at) - lse


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "attn": _run_attn, "logprobs": _run_logprobs}[state["kind"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------


def _exact_e4m3(x):
    """The e4m3 value nearest to x, ties to the even one: 3 bits behind the leading one, none below 2^-9."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(x / step) * step


def _exact_append(case, s):
    page, nkv = case["page"], case["nkv"]
    start, live, n = _plan(case)
    q_out = s["q_out"].double()
    kp, vp = s["k_pages"][LAYER].double(), s["v_pages"][LAYER].double().transpose(2, 3).contiguous()
    ks, vs = s["k_scale"][LAYER].double(), s["v_scale"][LAYER].double()
    table = s["table"].cpu()
    freq = torch.tensor([THETA ** (-i / 64.0) for i in range(64)], dtype=torch.float64, device=DEV)
    r0 = 0
    for b in range(case["nseq"]):
        if n[b] == 0:
            continue
        angle = torch.outer(torch.arange(start[b], start[b] + n[b], dtype=torch.float64, device=DEV), freq)
        rot = torch.polar(torch.ones_like(angle), angle)[:, None]

        def turned(x):
            z = torch.complex(x[..., :64].double(), x[..., 64:].double()) * rot
            return torch.cat((z.real, z.imag), dim=-1)

        sl = slice(r0, r0 + n[b])
        r0 += n[b]
        q_out[sl] = turned(s["q"][sl])
        kn, vn = turned(s["knew"][sl]), s["vnew"][sl].double()
        for j in range(start[b] // page, (start[b] + n[b] - 1) // page + 1):
            w0, w1 = max(start[b], j * page), min(start[b] + n[b], (j + 1) * page)
            end = min(live[b], (j + 1) * page)
            olds = [i - j * page for i in range(j * page, end) if not w0 <= i < w1]
            i = int(table[b, j])
            for new, pages, scale in ((kn, kp, ks), (vn, vp, vs)):
                x = new[w0 - start[b]:w1 - start[b]].transpose(0, 1)
                for h in range(nkv):
                    a = float(x[h].abs().max())
                    e = -100
                    if a > 0:
                        e = math.floor(math.log2(a / 448)) - 1
                        while a > 448 * 2.0 ** e:
                            e += 1
                        e = max(e, -100)
                    sc = 2.0 ** e
                    if olds:
                        was = float(scale[i, h])
                        if was >= sc:
                            sc = was
                        else:
                            at = torch.tensor(olds, device=DEV)
                            pages[i, h, at] = _exact_e4m3(pages[i, h, at] * (was / sc))
                    scale[i, h] = sc
                    pages[i, h, w0 - j * page:w1 - j * page] = _exact_e4m3(x[h] / sc)
    return q_out, kp, vp.transpose(2, 3).contiguous(), ks, vs


def _exact_attn(case, s):
    pre, total, n = _plan(case)
    nkv, group, page, b_ = case["nkv"], case["nq"] // case["nkv"], case["page"], case["mask"]
    out = s["q_out"].double()
    r0 = 0
    for b in range(case["nseq"]):
        if n[b] == 0:
            continue
        ids = s["table"][b, :-(-total[b] // page)].long()
        for h in range(nkv):
            k = (s["k_pages"][LAYER][ids, h].double() * s["k_scale"][LAYER][ids, h].double()[:, None, None]).reshape(-1, HD)[:total[b]]
            v = s["v_pages"][LAYER][ids, h].double() * s["v_scale"][LAYER][ids, h].double()[:, None, None]
            v = v.transpose(1, 2).reshape(-1, HD)[:total[b]]
            for c0 in range(0, n[b], 256):
                c1 = min(n[b], c0 + 256)
                q = s["q"][r0 + c0:r0 + c1, h * group:(h + 1) * group].double()
                sc = (q.reshape(-1, HD) @ k.T / math.sqrt(HD)).view(c1 - c0, group, -1)
                if b_:
                    end = (torch.arange(pre[b] + c0, pre[b] + c1, device=DEV) // b_ + 1) * b_
                    sc = sc.masked_fill(torch.arange(total[b], device=DEV)[None, None] >= end[:, None, None], -math.inf)
                out[r0 + c0:r0 + c1, h * group:(h + 1) * group] = (torch.softmax(sc, dim=-1).view(-1, total[b]) @ v).view(c1 - c0, group, HD)
        r0 += n[b]
    return out


def _exact_logprobs(case, s):
    parts = []
    for r in range(0, case["rows"], 64):
        x, ids = s["logits"][0, r:r + 64].double(), s["ids"][0, r:r + 64].long()
        lp = torch.log_softmax(x, dim=-1)
        ent = -torch.special.xlogy(lp.exp(), lp.exp()).sum(dim=-1)
        pick = torch.where(ids < 0, torch.zeros_like(ent), lp[torch.arange(len(ids), device=DEV), ids.clamp_min(0)])
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        parts.append((pick, ent, order, torch.gather(lp, 1, order)))
    pick, ent, order, alt = (torch.cat(p)[None] for p in zip(*parts))
    return pick, ent, order.to(torch.int32), alt


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    return _exact_attn(case, s) if case["kind"] == "attn" else _exact_logprobs(case, s)
