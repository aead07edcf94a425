"""The operators of a paged cache held in 4 bits, and of the heads that go into it, as cases that can be timed and compared.

A program that keeps its own projections norms and rotates its queries and keys (for the attention callbacks and
16-bit caches on their own, for the paged cache as the rows are appended), appends keys and values to a paged cache
of 4-bit values, attends over that cache, and reads rows of it back into 16 bits.  Heads, prefixes and block sizes are
the 1.5B configuration's and the benchmark's (12 query heads on 2 kv heads of 128, prefixes of 512 to 8192 rows, blocks
of 32 and sub-blocks of 8, 16 sequences with prefixes in [128, 1024], a context window of 32768), and generic ones
beside them.

Layout of one layer's pages: keys and values [pages, kv heads, page, 64] bytes, two e2m1 codes each, the lower dim in
the lower four bits.  Keys have one power of two (its exponent + 127 in 8 bits) for each block of 32 dims: that of slot s
and block b is entry [s / 16, s % 4, b, s / 4 % 4] of [pages, kv heads, page / 16, 4, 4, 4].  Values have one bfloat16
scale for each slot and head, [pages, kv heads, page].  Position p of a sequence is slot p % page of the page that its
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
BLOCK = 32  # dims of a key that share a scale
THETA = 1e6
EPS = 1e-6
WINDOW = 32768  # positions that the unscaled rotation is made for
LAYERS, LAYER = 2, 1  # the caches hold two layers; the calls take the second
TD = {"bfloat16": torch.bfloat16, "float16": torch.float16}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # of codes 0 .. 7; 8 more: negative

# a case's fields: `nq` / `nkv` heads; `rot` dims of a head that turn, in pairs of neighbours where `inter`, with the
# frequencies `scaled` by `factor`; `norm` whether heads are normed first; `page` tokens a page; `nseq` sequences, whose
# cached lengths before the call come from [lo, hi] with `lens`; `rows` new rows of each (up to that many where `ragged`);
# `mask` 0 none, else block-causal in blocks of that many positions (1: causal)


def listed():
    plain = dict(rot=128, inter=False, scaled="none", factor=1.0, norm=False)
    return [
        # one sequence's next token, its heads normed and rotated for the attention callback: latency
        dict(name="rotate_1", kind="rotate", nq=12, nkv=2, rows=1, lo=2079, hi=2079, lens=1, rot=128, inter=False,
             scaled="none", factor=1.0, norm=True, dtype="bfloat16"),
        # the rows of many prompts, part of each head turned in neighbouring pairs
        dict(name="rotate_2500", kind="rotate", nq=12, nkv=2, rows=2500, lo=0, hi=1023, lens=2, rot=64, inter=True,
             scaled="linear", factor=2.0, norm=False, dtype="float16"),
        # the longest prompt, positions beyond the window that the frequencies are for
        dict(name="rotate_8192", kind="rotate", nq=12, nkv=2, rows=8192, lo=30000, hi=120000, lens=3, rot=128, inter=False,
             scaled="yarn", factor=4.0, norm=True, dtype="bfloat16"),
        # one sequence's next token, once a layer: latency
        dict(name="append_1x1", kind="append", nq=12, nkv=2, page=32, nseq=1, lo=2079, hi=2079, lens=1, rows=1,
             ragged=False, dtype="bfloat16", **dict(plain, norm=True)),
        # prompts of many lengths appended in one call
        dict(name="append_ragged", kind="append", nq=12, nkv=2, page=64, nseq=24, lo=0, hi=700, lens=5, rows=509,
             ragged=True, dtype="float16", **plain),
        # the longest prompt
        dict(name="append_8192", kind="append", nq=12, nkv=2, page=32, nseq=1, lo=0, hi=0, lens=1, rows=8192,
             ragged=False, dtype="bfloat16", **dict(plain, norm=True)),
        # many sequences' contexts read back, to go on with 16-bit rows
        dict(name="read_16", kind="read", nq=12, nkv=2, page=32, nseq=16, lo=0, hi=0, lens=3, rows=1024, ragged=True,
             dtype="float16"),
        # a context that fills the window read back
        dict(name="read_32768", kind="read", nq=12, nkv=2, page=64, nseq=1, lo=0, hi=0, lens=1, rows=32768, ragged=False,
             dtype="bfloat16"),
        # one sequence's next token over an ordinary prompt: latency
        dict(name="attn_1x1_p2080", kind="attn", nq=12, nkv=2, page=32, nseq=1, lo=2079, hi=2079, lens=1, rows=1,
             mask=0, ragged=False, dtype="bfloat16"),
        # many sequences' blocks refined together
        dict(name="attn_16x32", kind="attn", nq=12, nkv=2, page=32, nseq=16, lo=128, hi=1024, lens=3, rows=32,
             mask=0, ragged=False, dtype="float16"),
        # many sequences' next tokens over long prompts: the cache's bytes
        dict(name="attn_64x1_p8192", kind="attn", nq=12, nkv=2, page=64, nseq=64, lo=1024, hi=8191, lens=7, rows=1,
             mask=1, ragged=False, dtype="bfloat16"),
        # the last part of a long prompt, block-causal
        dict(name="attn_2048_p8192", kind="attn", nq=12, nkv=2, page=32, nseq=1, lo=6144, hi=6144, lens=1, rows=2048,
             mask=32, ragged=False, dtype="bfloat16"),
    ]


def _log_size(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng: random.Random):
    kind = rng.choice(("rotate", "append", "read", "attn", "attn"))
    nq, nkv = rng.choice(((12, 2), (12, 2), (4, 2), (8, 8), (16, 1)))
    c = dict(kind=kind, nq=nq, nkv=nkv, dtype=rng.choice(("bfloat16", "bfloat16", "float16")), lens=rng.randrange(1 << 20))
    scaled = rng.choice(("none", "none", "linear", "ntk", "yarn"))
    turn = dict(rot=rng.choice((128, 128, 64, 32)), inter=rng.random() < 0.4, scaled=scaled,
                factor=1.0 if scaled == "none" else rng.choice((2.0, 4.0, 8.0)), norm=rng.random() < 0.5)
    if kind == "rotate":
        lo = _log_size(rng, 1, 100000)
        return dict(c, **turn, rows=_log_size(rng, 1, 8192), lo=lo, hi=lo + _log_size(rng, 1, 30000))
    c.update(page=rng.choice((16, 32, 32, 64, 128)), nseq=_log_size(rng, 1, 64), ragged=rng.random() < 0.3)
    if kind == "read":
        return dict(c, lo=rng.choice((0, 0, _log_size(rng, 1, 2000))), hi=2000, rows=_log_size(rng, 1, max(1, WINDOW // c["nseq"])))
    rows = rng.choice((1, 8, 32, _log_size(rng, 1, max(1, 4096 // c["nseq"]))))
    lo = _log_size(rng, 1, 8192 // c["nseq"] + 64)
    hi = lo + _log_size(rng, 1, 40000 // c["nseq"])
    if kind == "append":
        return dict(c, **turn, lo=lo, hi=hi, rows=rows)
    # (queries times keys are bounded by the largest listed case's)
    rows = max(1, min(rows, 200_000_000 // (c["nseq"] * nq * (hi + rows))))
    return dict(c, lo=lo, hi=hi, rows=rows, mask=rng.choice((0, 1, 32)))


# ---- what a case's sizes come to ---------------------------------------------------------------------------


def _plan(case):
    """Per sequence: first position of its rows, positions that it holds after the call, rows."""
    rng = random.Random(case["lens"])
    first = [rng.randint(case["lo"], case["hi"]) for _ in range(case["nseq"])]
    n = [rng.randint(0, case["rows"]) if case["ragged"] else case["rows"] for _ in first]
    if case["ragged"]:
        n[-1] = case["rows"]
    return first, [p + k for p, k in zip(first, n)], n


def _pairs(case):
    """(query row, key) pairs that the attention takes."""
    pre, total, n = _plan(case)
    b, pairs = case["mask"], 0
    for p, t, k in zip(pre, total, n):
        pairs += k * t if not b else sum(min(t, ((p + i) // b + 1) * b) for i in range(k))
    return pairs


ROW_BYTES = HD // 2 + 4 + HD // 2 + 2  # of a position and kv head: key, its scales, value, its scale


def work(case):
    nq, nkv = case["nq"], case["nkv"]
    if case["kind"] == "rotate":
        n = case["rows"] * (nq + nkv)
        return dict(bytes=n * HD * 4 + case["rows"] * 4, flops=n * (3 * case["rot"] + (4 * HD if case["norm"] else 0)))
    _, total, n = _plan(case)
    rows = sum(n)
    if case["kind"] == "read":
        return dict(bytes=rows * nkv * (ROW_BYTES + 4 * HD), flops=2 * rows * nkv * HD)
    if case["kind"] == "append":
        # q, k and v read, q written in 16 bits; k and v written in 4 and read back in 16
        return dict(bytes=rows * (4 * nq * HD + nkv * (4 * HD + 2 * ROW_BYTES + 4 * HD)),
                    flops=rows * ((nq + nkv) * (3 * case["rot"] + (4 * HD if case["norm"] else 0)) + 6 * nkv * HD))
    seen = sum(t for t, k in zip(total, n) if k)
    return dict(bytes=seen * nkv * ROW_BYTES + 4 * rows * nq * HD, flops=4 * HD * nq * _pairs(case))


# ---- inputs ------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _codes(x, scale):
    """The e2m1 codes nearest to x / scale, ties to the even one (borders times scale are exact in 64 bits)."""
    a = x.abs()
    code = torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a > border * scale) if i % 2 == 0 else (a >= border * scale)
    return code | (torch.signbit(x).to(torch.uint8) << 3)


def _packed(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _key_exponents(blocks):
    """The least e >= -60 with all of a block's values at most 7 x 2^e (7 = 0.875 x 2^3)."""
    m, e = torch.frexp(blocks.abs().amax(dim=-1).double())
    return torch.where(m > 0, e - 3 + (m > 0.875).to(e.dtype), -60).clamp(-60, 125)


def _value_scales(rows):
    """A sixth of the largest value, in bfloat16."""
    return (rows.abs().amax(dim=-1).double() / 6).float().to(torch.bfloat16).clamp_min(2.0 ** -60)


def _keys4(x):
    """Rows of keys [..., 128] as packed codes [..., 64] and exponents + 127 [..., 4]."""
    e = _key_exponents(x.unflatten(-1, (HD // BLOCK, BLOCK)))
    scale = torch.exp2(e.double()).to(x.dtype)
    return _packed(_codes(x, scale.repeat_interleave(BLOCK, dim=-1))), (e + 127).to(torch.uint8)


def _values4(x):
    s = _value_scales(x)
    return _packed(_codes(x, s.to(x.dtype)[..., None])), s


def _slots_in(x):
    """Scales of slots [..., page, 4] as they lie in a page: [..., page / 16, 4, 4, 4]."""
    return x.unflatten(-2, (-1, 4, 4)).movedim(-3, -1)


def _slots_out(x):
    """And back: [..., page / 16, 4, 4, 4] to [..., page, 4]."""
    return x.movedim(-1, -3).flatten(-4, -2)


def prepare(case, seed):
    g = _generator(seed)
    nq, nkv, td = case["nq"], case["nkv"], TD[case["dtype"]]
    s = dict(case)
    if case["kind"] in ("rotate", "append"):
        s["freq"] = _frequencies(case)
        for name in ("q_norm", "k_norm"):
            s[name] = (1.0 + _normal(g, (HD,), 0.2)).to(td) if case["norm"] else None
    if case["kind"] == "rotate":
        rows = case["rows"]
        rng = random.Random(case["lens"])
        at = rng.randint(case["lo"], case["hi"])
        # rows of one sequence or of several, each from where it stands
        pos = [at]
        while len(pos) < rows:
            pos.append(pos[-1] + 1 if rng.random() > 0.003 else rng.randint(case["lo"], case["hi"]))
        qkv = _normal(g, (rows, (nq + 2 * nkv) * HD)) * torch.exp(_normal(g, (rows, 1), 0.5))
        heads = qkv.to(td).view(rows, nq + 2 * nkv, HD)
        return dict(s, q=heads[:, :nq], k=heads[:, nq:nq + nkv], pos=_i32(pos),
                    q_out=torch.zeros((rows, nq, HD), dtype=td, device=DEV),
                    k_out=torch.zeros((rows, nkv, HD), dtype=td, device=DEV))
    page, nseq = case["page"], case["nseq"]
    a, total, n = _plan(case)
    rows = sum(n) + (3 if case["ragged"] else 0)  # ragged batches come padded
    need = [max(1, -(-t // page)) for t in total]
    width, pool = max(need) + 1, sum(need) + 2
    perm = torch.randperm(pool, generator=g, device=DEV).to(torch.int32).tolist()
    table = torch.full((nseq, width), -1, dtype=torch.int32)
    live = torch.zeros((pool, page), dtype=torch.bool)
    at = 0
    for b in range(nseq):
        ids = torch.tensor(perm[at:at + need[b]], dtype=torch.int32)
        at += need[b]
        table[b, :need[b]] = ids
        live[ids.long()] = torch.arange(need[b] * page).view(need[b], page) < total[b]
    live = live.to(DEV)[:, None, :]
    # slots that are not live hold what earlier owners of the page left there: scales that are NaN among it
    kc, ke = _keys4(_normal(g, (pool, nkv, page, HD)) * torch.exp(_normal(g, (nkv, 1, HD), 0.4)))
    vc, vs = _values4(_normal(g, (pool, nkv, page, HD), 0.7))
    ke = torch.where(live[..., None], ke, 255)
    vs = torch.where(live, vs, math.nan)
    k, v = (torch.zeros((LAYERS, *x.shape), dtype=torch.uint8, device=DEV) for x in (kc, vc))
    k[:], v[:] = kc, vc
    k_scale = _slots_in(ke)[None].repeat(LAYERS, 1, 1, 1, 1, 1, 1).contiguous()
    v_scale = vs[None].repeat(LAYERS, 1, 1, 1).contiguous()
    starts = [0]
    for c in n:
        starts.append(starts[-1] + c)
    s.update(k_codes=k, v_codes=v, k_scale=k_scale, v_scale=v_scale, table=table.to(DEV), max_rows=max(n), count=rows,
             row_start=_i32(starts) if case["ragged"] else None, start=_i32(a))
    if case["kind"] != "attn":
        for name in ("k_back", "v_back"):
            s[name] = torch.zeros((rows, nkv, HD), dtype=td, device=DEV)
        if case["kind"] == "read":
            return s
    # the projections of a step: one fused [q | k | v] row each, queries and keys before their rotation
    qkv = _normal(g, (rows, (nq + 2 * nkv) * HD)) * torch.exp(_normal(g, (rows, 1), 0.5))
    s["q_out"] = torch.zeros((rows, nq, HD), dtype=td, device=DEV)
    if case["kind"] == "append":
        heads = qkv.to(td).view(rows, nq + 2 * nkv, HD)
        return dict(s, q=heads[:, :nq], knew=heads[:, nq:nq + nkv], vnew=heads[:, nq + nkv:])
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

    cfg = FastDLLMConfig(vocab_size=256, hidden_size=128, intermediate_size=128, num_hidden_layers=LAYERS, rms_norm_eps=EPS,
                         num_attention_heads=nq, num_key_value_heads=nkv, head_dim=HD, rope_theta=THETA)
    shapes = param_shapes(cfg)
    return HipVM(cfg, [torch.zeros(shapes[n], dtype=TORCH_DTYPES[dtype], device=DEV) for n in param_names(cfg)], dtype=dtype)


@functools.lru_cache(maxsize=None)
def _rotary(rot, inter, scaled, factor):
    """The positions' plan that a program keeps."""
    from fast_dllm_relax_amd.rotary import Rotary

    scaling = None if scaled == "none" else dict(type=scaled, factor=factor)
    if scaled == "yarn":
        scaling["original_len"] = WINDOW
    return Rotary(theta=THETA, dim=rot, interleaved=inter, scaling=scaling)


def _cache(s):
    """The cache object that a program makes once over its pages."""
    if "cache" not in s:
        from fast_dllm_relax_amd.paged4 import Paged4KVCache

        s["cache"] = Paged4KVCache(k=s["k_codes"], v=s["v_codes"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s["cache"]


def _run_own(s):
    vm = _vm(s["dtype"], s["nq"], s["nkv"])
    if s["kind"] == "rotate":
        rotary = _rotary(s["rot"], s["inter"], s["scaled"], s["factor"])
        return vm.rotate_heads(s["q"], s["k"], s["pos"], rotary=rotary, q_norm=s["q_norm"], k_norm=s["k_norm"],
                               q_out=s["q_out"], k_out=s["k_out"])
    more = dict(row_start=s["row_start"], max_rows=s["max_rows"])
    if s["kind"] == "attn":
        return vm.paged_attn(s["q"], _cache(s), LAYER, s["table"], s["kv_len"], mask_block=s["mask"], out=s["q_out"], **more)
    back = dict(k_out=s["k_back"], v_out=s["v_back"], **more)
    if s["kind"] == "read":
        return vm.paged4_read(_cache(s), LAYER, s["table"], s["start"], s["count"], **back)
    rotary = _rotary(s["rot"], s["inter"], s["scaled"], s["factor"])
    q = vm.paged4_append(s["knew"], s["vnew"], _cache(s), LAYER, s["table"], s["start"], q=s["q"], q_out=s["q_out"],
                         rotary=rotary, q_norm=s["q_norm"], k_norm=s["k_norm"], **more)
    # what the cache now holds of these rows
    k, v = vm.paged4_read(_cache(s), LAYER, s["table"], s["start"], s["count"], **back)
    return q, k, v


# ---- the plain forms ---------------------------------------------------------------------------------------


def _frequencies(case):
    """Radians a position of each pair, and the factor of the turned dims (64 bits, [rot / 2])."""
    rot, factor = case["rot"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    theta = THETA * factor ** (rot / (rot - 2)) if case["scaled"] == "ntk" else THETA
    freq, gain = theta ** (-2 * i / rot), 1.0
    if case["scaled"] == "linear":
        freq = freq / factor
    if case["scaled"] == "yarn":
        # pairs that turn often in the window keep their frequency, those that turn less than once are slowed
        pair = [rot * math.log(WINDOW / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
        slow = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        freq, gain = freq * (1 - slow) + freq / factor * slow, 0.1 * math.log(factor) + 1
    return freq.to(DEV), gain


def _plain_turn(s, x, pos, weight):
    """x [n, heads, 128] normed and turned by positions pos [n], in 64 bits (far positions' angles need them)."""
    x = x.double()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * weight.double()
    freq, gain = s["freq"]
    angle = pos.double()[:, None] * freq
    c, n = (gain * f(angle)[:, None] for f in (torch.cos, torch.sin))
    rot = s["rot"]
    head, rest = x[..., :rot], x[..., rot:]
    if s["inter"]:
        x1, x2 = head[..., 0::2], head[..., 1::2]
        head = torch.stack((x1 * c - x2 * n, x2 * c + x1 * n), dim=-1).flatten(-2)
    else:
        x1, x2 = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat((x1 * c - x2 * n, x2 * c + x1 * n), dim=-1)
    return torch.cat((head, rest), dim=-1)


def _run_rotate(s):
    s["q_out"][:] = _plain_turn(s, s["q"], s["pos"], s["q_norm"]).to(s["q_out"].dtype)
    s["k_out"][:] = _plain_turn(s, s["k"], s["pos"], s["k_norm"]).to(s["k_out"].dtype)
    return s["q_out"], s["k_out"]


def _spread(s):
    """Index of each sequence's row i among the call's rows, [nseq, max_rows], and which of them there are."""
    i = torch.arange(s["max_rows"], device=DEV)[None]
    if s["row_start"] is None:
        at = torch.arange(s["nseq"], device=DEV)[:, None] * s["max_rows"] + i
        return at, torch.ones_like(at, dtype=torch.bool)
    first, last = s["row_start"][:-1, None], s["row_start"][1:, None]
    return (first + i).clamp_max(s["count"] - 1), first + i < last


def _places(s):
    """Of the rows that there are: index among the call's, position, page and slot."""
    at, there = _spread(s)
    pos = (s["start"][:, None] + torch.arange(s["max_rows"], device=DEV)[None])[there]
    seq = torch.arange(s["nseq"], device=DEV)[:, None].expand_as(at)[there]
    return at[there], pos, s["table"][seq, pos // s["page"]].long(), pos % s["page"]


@functools.lru_cache(maxsize=None)
def _values():
    return torch.tensor([*VALUES, *(-v for v in VALUES)], device=DEV)


def _unpacked(code):
    """Packed codes [..., n] as the values they stand for [..., 2 n]."""
    return _values()[torch.stack((code & 15, code >> 4), dim=-1).flatten(-2).long()]


def _key_scales(e):
    return torch.where(e == 255, math.nan, torch.exp2(e.float() - 127))


def _run_read(s):
    at, _, page, slot = _places(s)
    e = s["k_scale"][LAYER][page, :, slot // 16, slot % 4, :, slot // 4 % 4]
    k = _unpacked(s["k_codes"][LAYER][page, :, slot]) * _key_scales(e).repeat_interleave(BLOCK, dim=-1)
    v = _unpacked(s["v_codes"][LAYER][page, :, slot]) * s["v_scale"][LAYER][page, :, slot].float()[..., None]
    s["k_back"][at] = k.to(s["k_back"].dtype)
    s["v_back"][at] = v.to(s["v_back"].dtype)
    return s["k_back"], s["v_back"]


def _run_append(s):
    at, pos, page, slot = _places(s)
    s["q_out"][at] = _plain_turn(s, s["q"][at], pos, s["q_norm"]).to(s["q_out"].dtype)
    code, e = _keys4(_plain_turn(s, s["knew"][at], pos, s["k_norm"]))
    s["k_codes"][LAYER][page, :, slot] = code
    s["k_scale"][LAYER][page, :, slot // 16, slot % 4, :, slot // 4 % 4] = e
    code, scale = _values4(s["vnew"][at].double())
    s["v_codes"][LAYER][page, :, slot] = code
    s["v_scale"][LAYER][page, :, slot] = scale
    return s["q_out"], *_run_read(s)


def _run_attn(s):
    nq, nkv, page, nseq = s["nq"], s["nkv"], s["page"], s["nseq"]
    group, width = nq // nkv, s["table"].shape[1]
    at, there = _spread(s)
    keys = torch.arange(width * page, device=DEV)
    live = keys[None] < s["kv_len"][:, None]
    ids = s["table"].clamp_min(0).long()
    scale = _key_scales(_slots_out(s["k_scale"][LAYER][ids])).repeat_interleave(BLOCK, dim=-1)
    k = (_unpacked(s["k_codes"][LAYER][ids]) * scale).permute(0, 2, 1, 3, 4).reshape(nseq, nkv, width * page, HD)
    v = _unpacked(s["v_codes"][LAYER][ids]) * s["v_scale"][LAYER][ids].float()[..., None]
    v = v.permute(0, 2, 1, 3, 4).reshape(nseq, nkv, width * page, HD)
    k = torch.where(live[:, None, :, None], k, 0.0)
    v = torch.where(live[:, None, :, None], v, 0.0)
    q = s["q"][at].float().view(nseq, s["max_rows"], nkv, group, HD).permute(0, 2, 1, 3, 4)
    q = q.reshape(nseq, nkv, s["max_rows"] * group, HD)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(HD))
    pos = (s["kv_len"] - there.sum(dim=1))[:, None] + torch.arange(s["max_rows"], device=DEV)[None]
    see = live[:, None, :].expand(nseq, s["max_rows"], width * page)
    if s["mask"]:
        see = see & (keys[None, None] < ((pos // s["mask"] + 1) * s["mask"])[:, :, None])
    score = torch.where(see[:, None, :, None], score.view(nseq, nkv, s["max_rows"], group, -1), -math.inf)
    p = torch.exp(score - score.amax(dim=-1, keepdim=True).clamp_min(-1e30))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(nseq, nkv, s["max_rows"] * group, -1), v).view(nseq, nkv, s["max_rows"], group, HD)
    o = o.permute(0, 2, 1, 3, 4).reshape(nseq, s["max_rows"], nq, HD)
    s["q_out"][at[there]] = o[there].to(s["q_out"].dtype)
    return s["q_out"]


def run(state):
    if own:
        return _run_own(state)
    return {"rotate": _run_rotate, "append": _run_append, "read": _run_read, "attn": _run_attn}[state["kind"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------


def _exact_turn(case, x, positions, weight):
    """Heads as complex pairs times e^(i angle); the frequencies once more, from their definition."""
    rot, f = case["rot"], case["factor"]
    theta = THETA * f ** (rot / (rot - 2.0)) if case["scaled"] == "ntk" else THETA
    freq, gain = [], 1.0
    for i in range(rot // 2):
        w = math.exp(-2 * i / rot * math.log(theta))
        if case["scaled"] == "linear":
            w /= f
        elif case["scaled"] == "yarn":
            edges = [rot / 2 * math.log(WINDOW / (2 * math.pi * t), theta) for t in (32, 1)]
            lo, hi = max(0, math.floor(edges[0])), min(rot - 1, math.ceil(edges[1]))
            mix = min(1.0, max(0.0, (i - lo) / (hi - lo if hi > lo else 0.001)))
            w = w * (1 - mix) + w / f * mix
            gain = 1 + math.log(f) / 10
        freq.append(w)
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / HD + EPS).sqrt() * weight.double()
    angle = torch.outer(positions.double(), torch.tensor(freq, dtype=torch.float64, device=DEV))
    pairs = x[..., :rot].unflatten(-1, (rot // 2, 2) if case["inter"] else (2, rot // 2))
    if not case["inter"]:
        pairs = pairs.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, gain), angle)[:, None])
    if not case["inter"]:
        turned = turned.transpose(-1, -2)
    return torch.cat((turned.flatten(-2), x[..., rot:]), dim=-1)


def _exact_e2m1(x):
    """The value of (1 + m / 2) 2^e, e in 0 .. 2, or of m / 2, that is nearest to x, ties to the even m; 6 at most."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(0, 2).double() - 1)
    return (torch.round(x / step) * step).clamp(-6, 6)


def _exact_keys(x):
    amax = x.abs().unflatten(-1, (-1, BLOCK)).amax(-1)
    e = torch.ceil(torch.log2(amax / 7)) - 1
    for _ in range(2):
        e = torch.where(amax > 7 * torch.exp2(e), e + 1, e)
    scale = torch.exp2(e.clamp(-60, 125)).repeat_interleave(BLOCK, -1)
    return _exact_e2m1(x / scale) * scale


def _exact_values(x):
    scale = (x.abs().amax(-1, keepdim=True) / 6).to(torch.bfloat16).double().clamp_min(2.0 ** -60)
    return _exact_e2m1(x / scale) * scale


def _exact_held(case, s, b, lo, hi):
    """What sequence b's positions [lo, hi) of the cache hold."""
    page = case["page"]
    pos = torch.arange(lo, hi, device=DEV)
    pg, slot = s["table"][b].long()[pos // page], pos % page
    out = []
    for codes in (s["k_codes"][LAYER][pg, :, slot], s["v_codes"][LAYER][pg, :, slot]):
        c = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2).long()
        e, m = (c % 8) // 2, (c % 2).double()
        size = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1))
        out.append(torch.where(c >= 8, -size, size))
    e = s["k_scale"][LAYER][pg, :, slot // 16, slot % 4, :, (slot % 16) // 4].double()
    return out[0] * torch.exp2(e - 127).repeat_interleave(BLOCK, -1), out[1] * s["v_scale"][LAYER][pg, :, slot].double()[..., None]


def _exact_append(case, s):
    first, _, n = _plan(case)
    q, k, v = s["q_out"].double(), s["k_back"].double(), s["v_back"].double()
    r0 = 0
    for b in range(case["nseq"]):
        sl = slice(r0, r0 + n[b])
        r0 += n[b]
        if n[b]:
            at = torch.arange(first[b], first[b] + n[b], device=DEV)
            q[sl] = _exact_turn(case, s["q"][sl], at, s["q_norm"])
            k[sl] = _exact_keys(_exact_turn(case, s["knew"][sl], at, s["k_norm"]))
            v[sl] = _exact_values(s["vnew"][sl].double())
    return q, k, v


def _exact_read(case, s):
    first, total, n = _plan(case)
    k, v = s["k_back"].double(), s["v_back"].double()
    r0 = 0
    for b in range(case["nseq"]):
        if n[b]:
            k[r0:r0 + n[b]], v[r0:r0 + n[b]] = _exact_held(case, s, b, first[b], total[b])
        r0 += n[b]
    return k, v


def _exact_attn(case, s):
    pre, total, n = _plan(case)
    group, mask = case["nq"] // case["nkv"], case["mask"]
    out = s["q_out"].double()
    r0 = 0
    for b in range(case["nseq"]):
        if n[b] == 0:
            continue
        keys, values = _exact_held(case, s, b, 0, total[b])
        for h in range(case["nkv"]):
            k, v = keys[:, h], values[:, h]
            for c0 in range(0, n[b], 256):
                c1 = min(n[b], c0 + 256)
                q = s["q"][r0 + c0:r0 + c1, h * group:(h + 1) * group].double()
                sc = (q.reshape(-1, HD) @ k.T / math.sqrt(HD)).view(c1 - c0, group, -1)
                if mask:
                    end = (torch.arange(pre[b] + c0, pre[b] + c1, device=DEV) // mask + 1) * mask
                    sc = sc.masked_fill(torch.arange(total[b], device=DEV)[None, None] >= end[:, None, None], -math.inf)
                out[r0 + c0:r0 + c1, h * group:(h + 1) * group] = (torch.softmax(sc, dim=-1).view(-1, total[b]) @ v).view(c1 - c0, group, HD)
        r0 += n[b]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotate":
        return tuple(_exact_turn(case, s[x], s["pos"], s[x + "_norm"]) for x in ("q", "k"))
    return {"append": _exact_append, "read": _exact_read, "attn": _exact_attn}[case["kind"]](case, s)
