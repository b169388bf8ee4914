"""Cases for timing the decode-side operators of the latent cache: the MXFP8 cache written and read back, attention of a
batch that shares a long prefix over it, and the verification of drafted tokens.

`listed()` and `draw(rng)` give cases (plain dicts), `prepare(case, seed)` makes one case's inputs on the GPU, and
`run(state)` makes one pass.  With `own` false the pass is the operators' plain form: elementary torch operations in 32 bits
(64 for the sums that a sampled token depends on).  With `own` true it is the library's entry points through the binding.
`exact(case, seed)` evaluates the definition in 64 bits, `work(case)` counts the bytes and operations no form can do without.

Cache pages hold 64 tokens of one layer.  An MXFP8 page is 41984 bytes: 64 x 512 E4M3 codes, 64 x 64 bf16 (the part that
is not normalised), 64 x 16 UE8M0 scale bytes, one for each 32 codes.  A bf16 page is 64 rows of 576.
"""
import math
import os
import sys

import torch

own = False

PAGE, LATENT, ROPE, ROW = 64, 512, 64, 576
CODES, ROPE_AT, SCALES_AT, MX8_PAGE = PAGE * LATENT, PAGE * LATENT, PAGE * LATENT + PAGE * ROPE * 2, 41984
LAYERS = 2                      # two layers share a page, as a model's layers do: the measured one is the second
SOFTMAX_SCALE = 192 ** -0.5
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the new tokens of one decode step of a batch, rows taken out of the projection's 2112 columns
        {"name": "store decode step", "op": "store", "tokens": 96, "stride": 2112},
        # the whole prompt of a 16k prefill, one row short of full pages
        {"name": "store 16k prompt", "op": "store", "tokens": 16383, "stride": 576},
        # a short cached prompt read back before its continuation is prefilled
        {"name": "gather short prompt", "op": "gather", "tokens": 700, "rows": 768},
        # a long cached prompt read back
        {"name": "gather 64k prompt", "op": "gather", "tokens": 65500, "rows": 65536},
        # a single user's next token: the smallest call, latency alone
        {"name": "attn one sequence", "op": "attn", "batch": 1, "steps": 1, "heads": 24, "prefix": 0, "longest": 500, "mx8": True},
        # a chat batch behind one system prompt
        {"name": "attn chat batch", "op": "attn", "batch": 32, "steps": 1, "heads": 24, "prefix": 8229, "longest": 1024, "mx8": True},
        # the same batch verifying three drafted tokens and the one after
        {"name": "attn drafted tokens", "op": "attn", "batch": 48, "steps": 4, "heads": 24, "prefix": 16384, "longest": 512, "mx8": True},
        # half the heads on one card, bf16 pages as the prompt pass leaves them
        {"name": "attn bf16 pages", "op": "attn", "batch": 16, "steps": 2, "heads": 48, "prefix": 4000, "longest": 2048, "mx8": False},
        # questions to one very long document, all heads on one card
        {"name": "attn long document", "op": "attn", "batch": 8, "steps": 1, "heads": 96, "prefix": 131072, "longest": 250, "mx8": True},
        # unrelated conversations, nothing shared: bound by the cache's bytes
        {"name": "attn no shared prefix", "op": "attn", "batch": 64, "steps": 1, "heads": 12, "prefix": 0, "longest": 4096, "mx8": True},
        # one sequence, drafts from a lookup (no probabilities of their own)
        {"name": "verify one lookup draft", "op": "verify", "batch": 1, "steps": 5, "vocab": 163840, "probs": False},
        # a batch of drafts sampled from a small model
        {"name": "verify draft batch", "op": "verify", "batch": 64, "steps": 4, "vocab": 163840, "probs": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "gather", "attn", "attn", "attn", "verify"])
    if op == "store":
        return {"op": op, "tokens": _log(rng, 1, 16383), "stride": rng.choice([576, 584, 2112])}
    if op == "gather":
        rows = _log(rng, 1, 65536)
        return {"op": op, "tokens": rng.randint(0, rows), "rows": rows}
    if op == "verify":
        return {"op": op, "batch": _log(rng, 1, 64), "steps": rng.randint(1, 4), "vocab": _log(rng, 1000, 163840), "probs": rng.random() < 0.7}
    batch, steps, heads = _log(rng, 1, 64), rng.choice([1, 1, 2, 3, 4, 6]), rng.choice([5, 12, 16, 24, 48, 96])
    most = 8 * 96 * 131072 // (batch * steps * heads)          # no more scores than the long document's
    longest = _log(rng, steps, max(steps, min(4096, most, 262144 // batch)))
    prefix = 0 if rng.random() < 0.2 else _log(rng, 1, max(1, min(131072, most - longest)))
    return {"op": "attn", "batch": batch, "steps": steps, "heads": heads, "prefix": prefix, "longest": longest, "mx8": rng.random() < 0.7}


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _suffix_lens(case):
    """Tokens in each sequence's own pages, its new ones included: spread from a few to the longest, one at the longest."""
    b, s, top = case["batch"], case["steps"], case["longest"]
    return [top if i == 0 else s + i * 7919 % (top - s + 1) for i in range(b)]


# ---- the cache in plain torch -------------------------------------------------------------------------------------------
def _planes(cache):
    """(codes, rope, scales) of the measured layer of an MXFP8 cache [pages, LAYERS, 41984], as views."""
    p = cache[:, 1]
    n = p.shape[0]
    return (p[:, :CODES].view(torch.float8_e4m3fn).view(n, PAGE, LATENT), p[:, ROPE_AT:SCALES_AT].view(BF16).view(n, PAGE, ROPE),
            p[:, SCALES_AT:].view(n, PAGE, LATENT // 32))


def _quantise(x):
    """[n, 512] bf16 -> (codes, scale bytes): e is the smallest whole number with 448 * 2^e >= the block's largest magnitude."""
    blocks = x.float().view(-1, LATENT // 32, 32)
    man, exp = torch.frexp(blocks.abs().amax(-1) / 448.0)       # amax / 448 = man * 2^exp with man in [0.5, 1)
    # the quotient is rounded in 32 bits, but a bf16 other than 448 * 2^k is 1/224 or more away from it: man == 0.5 means equal
    e = torch.where(man == 0, 0, torch.where(man == 0.5, exp - 1, exp)).clamp(-127, 127)
    codes = torch.ldexp(blocks, -e[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(-1, LATENT), (e + 127).to(torch.uint8)


def _read(st, table, dtype):
    """The cached rows [..., 64 * pages, 576] of a block table, as numbers of `dtype`."""
    shape = list(table.shape[:-1]) + [table.shape[-1] * PAGE]
    if not st["mx8"]:
        return st["cache"][:, 1][table.long()].reshape(shape + [ROW]).to(dtype)
    codes, rope, scales = (p[table.long()] for p in (_planes(st["cache"])[0].view(torch.uint8), *_planes(st["cache"])[1:]))
    lat = codes.view(torch.float8_e4m3fn).to(dtype).reshape(shape + [LATENT // 32, 32])
    lat = lat * torch.exp2(scales.to(dtype) - 127).reshape(shape + [LATENT // 32, 1])
    return torch.cat([lat.reshape(shape + [LATENT]), rope.reshape(shape + [ROPE]).to(dtype)], -1)


# ---- inputs -------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed) * 2 + 1)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    st = dict(case)
    if case["op"] == "verify":
        b, s, v = case["batch"], case["steps"], case["vocab"]
        logits = normal(b, s + 1, v) * 2.5
        st["target"] = torch.softmax(logits, -1)
        draft = torch.softmax(logits[:, :s] + 0.5 * normal(b, s, v), -1)
        st["ids"] = torch.multinomial(draft.view(b * s, v), 1, generator=g).view(b, s) if case["probs"] else logits[:, :s].argmax(-1)
        st["draft"] = draft if case["probs"] else None
        st["u"] = torch.rand((b, s + 1), generator=g, device=dev)
        st["accepted"] = torch.empty(b, dtype=torch.int32, device=dev)
        st["tokens"] = torch.empty((b, s + 1), dtype=torch.int64, device=dev)
        return st

    if case["op"] == "store":
        n, pages = case["tokens"], _pages(case["tokens"]) + 1
        st["rows"] = normal(n, case["stride"]).to(BF16)
        st["slots"] = torch.randperm(pages, generator=g, device=dev).view(-1, 1).mul(PAGE).add(torch.arange(PAGE, device=dev)).view(-1)[:n].contiguous()
        st["cache"] = torch.zeros((pages, LAYERS, MX8_PAGE), dtype=torch.uint8, device=dev)
        return st

    lens = [case["tokens"]] if case["op"] == "gather" else _suffix_lens(case)
    shared = 0 if case["op"] == "gather" else case["prefix"]
    width = _pages(case["rows"]) if case["op"] == "gather" else _pages(max(lens))
    used = [_pages(n) for n in lens]
    pages = _pages(shared) + (width if case["op"] == "gather" else sum(used)) + 1
    st["mx8"] = case.get("mx8", True)
    rows = normal(pages * PAGE, ROW).to(BF16)
    if st["mx8"]:
        st["cache"] = torch.zeros((pages, LAYERS, MX8_PAGE), dtype=torch.uint8, device=dev)
        codes, rope, scales = _planes(st["cache"])
        c, e = _quantise(rows[:, :LATENT])
        codes.view(torch.uint8).copy_(c.view(torch.uint8).view(pages, PAGE, LATENT))
        rope.copy_(rows[:, LATENT:].reshape(pages, PAGE, ROPE))
        scales.copy_(e.view(pages, PAGE, LATENT // 32))
    else:
        st["cache"] = torch.zeros((pages, LAYERS, PAGE, ROW), dtype=BF16, device=dev)
        st["cache"][:, 1] = rows.view(pages, PAGE, ROW)
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    at = _pages(shared)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    if case["op"] == "gather":
        st["table"] = order[:width].contiguous()
        st["out"] = torch.empty((case["rows"], ROW), dtype=BF16, device=dev)
        return st
    st["prefix_table"] = order[:max(1, at)].contiguous()
    st["prefix_len"] = torch.tensor([shared], dtype=torch.int32, device=dev)
    first = torch.tensor([at + sum(used[:i]) for i in range(len(used))], device=dev)
    column = torch.arange(width, device=dev)
    own_page = column[None] < torch.tensor(used, device=dev)[:, None]
    st["table"] = torch.where(own_page, order[(first[:, None] + column[None]).clamp(max=pages - 1)], 0).to(torch.int32).contiguous()
    b, s, h = case["batch"], case["steps"], case["heads"]
    st["q"] = (1.4 * normal(b, s, h, ROW)).to(BF16)
    st["out"] = torch.empty((b, s, h, LATENT), dtype=BF16, device=dev)
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------
def _k3g():
    at = os.path.join(os.getcwd(), "kern-k3_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import k3g
    return k3g


def run(st):
    if own:
        return _run_own(st, _k3g())
    return {"store": _store, "gather": _gather, "attn": _attn, "verify": _verify}[st["op"]](st)


def _run_own(st, k3g):
    s = k3g.current_stream()
    if st["op"] == "verify":
        k3g.call("k3g_verify_draft", st["target"], st["vocab"], st["draft"], st["vocab"], st["ids"], st["u"], st["accepted"], st["tokens"],
                 st["batch"], st["steps"], st["vocab"], s)
        return {"accepted": st["accepted"], "tokens": st["tokens"]}
    cache = st["cache"]
    if st["op"] == "store":
        k3g.call("k3g_latent_mx8_store", st["rows"], st["stride"], st["slots"], cache, MX8_PAGE, LAYERS * MX8_PAGE, cache.shape[0], st["tokens"], s)
        return dict(zip(("codes", "rope", "scales"), _planes(cache)))
    if st["op"] == "gather":
        k3g.call("k3g_latent_mx8_gather", cache, st["table"], MX8_PAGE, LAYERS * MX8_PAGE, cache.shape[0], st["lens"], st["out"], st["rows"], s)
        return st["out"]
    layer = MX8_PAGE if st["mx8"] else PAGE * ROW
    if "workspace" not in st:                                    # kept by the program, as its other buffers
        st["workspace"] = torch.empty(k3g.latent_attn_workspace(st["batch"], st["steps"], st["heads"]), dtype=torch.uint8, device=cache.device)
    k3g.call("k3g_latent_attn", st["q"], st["heads"] * ROW, cache, int(st["mx8"]), layer, LAYERS * layer, cache.shape[0], st["prefix_table"],
             st["prefix_len"], _pages(st["prefix"]), st["table"], st["lens"], st["table"].shape[1], st["out"], st["workspace"],
             st["workspace"].numel(), st["batch"], st["steps"], st["heads"], SOFTMAX_SCALE, s)
    return st["out"]


def _store(st):
    codes, rope, scales = _planes(st["cache"])
    page, at = st["slots"] // PAGE, st["slots"] % PAGE
    c, e = _quantise(st["rows"][:, :LATENT].contiguous())
    codes.view(torch.uint8)[page, at] = c.view(torch.uint8)
    rope[page, at] = st["rows"][:, LATENT:ROW]
    scales[page, at] = e
    return {"codes": codes, "rope": rope, "scales": scales}


def _gather(st):
    rows = _read(st, st["table"], F32)[:st["rows"]]
    live = torch.arange(st["rows"], device=rows.device) < st["lens"][0]
    st["out"].copy_(torch.where(live[:, None], rows, 0.0))
    return st["out"]


def _attn_of(st, dtype):
    """softmax(scale * q k^T) v over the shared prefix and each sequence's own tokens; v is the first 512 columns of k.  The
    token of step i sees the prefix and all but the last steps - 1 - i of its sequence's own tokens."""
    b, s, h = st["batch"], st["steps"], st["heads"]
    q = st["q"].to(dtype).view(b, s * h, ROW) * SOFTMAX_SCALE
    shared, tail = _read(st, st["prefix_table"], dtype), _read(st, st["table"], dtype)
    sp = (q.view(b * s * h, ROW) @ shared.T).view(b, s * h, -1)
    sp = torch.where(torch.arange(shared.shape[0], device=q.device) < st["prefix_len"], sp, -math.inf)
    ss = torch.bmm(q, tail.transpose(1, 2))
    step = torch.arange(s, device=q.device).repeat_interleave(h)
    seen = st["lens"].view(b, 1, 1) - (s - 1 - step).view(1, -1, 1)
    ss = torch.where(torch.arange(tail.shape[1], device=q.device) < seen, ss, -math.inf)
    top = torch.maximum(sp.amax(-1), ss.amax(-1))[..., None]
    top = torch.where(top == -math.inf, 0.0, top)
    sp, ss = torch.exp(sp - top), torch.exp(ss - top)
    total = sp.sum(-1) + ss.sum(-1)
    out = (sp.view(b * s * h, -1) @ shared[:, :LATENT]).view(b, s * h, LATENT) + torch.bmm(ss, tail[..., :LATENT])
    return torch.where(total[..., None] > 0, out / total[..., None], 0.0).view(b, s, h, LATENT)


def _attn(st):
    return _attn_of(st, F32).to(BF16)


def _verify(st):
    """Draft i is kept while u_i q_i(x_i) < p_i(x_i); the token after the last kept one is drawn from max(p - q, 0) if a draft
    was turned down there, else from p: the first v whose running sum passes u times the whole."""
    target, ids, u = st["target"], st["ids"], st["u"].to(F64)
    b, s, v = st["batch"], st["steps"], st["vocab"]
    px = target[:, :s].gather(-1, ids[..., None])[..., 0].to(F64)
    qx = st["draft"].gather(-1, ids[..., None])[..., 0].to(F64) if st["draft"] is not None else 1.0
    kept = (u[:, :s] * qx < px).long().cumprod(1).sum(1)
    lane = torch.arange(b, device=ids.device)
    p = target[lane, kept].to(F64)
    at = kept.clamp(max=s - 1)
    if st["draft"] is not None:
        q = st["draft"][lane, at].to(F64)
    else:
        q = (torch.arange(v, device=ids.device) == ids[lane, at][:, None]).to(F64)
    w = torch.where((kept < s)[:, None], (p - q).clamp(min=0.0), p)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p)
    c = w.cumsum(-1)
    pick = torch.searchsorted(c, u[:, s:] * c[:, -1:], right=True)
    last = torch.where(w > 0, torch.arange(v, device=ids.device), -1).amax(-1, keepdim=True)
    pick = torch.minimum(pick, last)
    column = torch.arange(s + 1, device=ids.device)
    drafted = torch.cat([ids, pick], 1)
    tokens = torch.where(column < kept[:, None], drafted, torch.where(column == kept[:, None], pick, -1))
    return {"accepted": kept.to(torch.int32), "tokens": tokens}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "verify":
        return None                                              # whole numbers
    st = prepare(case, seed)
    if case["op"] == "gather":
        rows = _exact_rows(st, st["table"])[:case["rows"]]
        rows[case["tokens"]:] = 0
        return rows
    if case["op"] == "attn":
        return _exact_attn(st)
    x = st["rows"][:, :LATENT].to(F64).view(-1, LATENT // 32, 32)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), 0.0).clamp(min=-127)
    y = x * torch.exp2(-e)
    grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)          # E4M3: three fraction bits, normal from 2^-6 up
    y = (torch.round(y / grid) * grid).clamp(-448, 448)
    pages = st["cache"].shape[0]
    codes = torch.zeros((pages * PAGE, LATENT), dtype=F64, device=x.device)
    rope = torch.zeros((pages * PAGE, ROPE), dtype=F64, device=x.device)
    codes[st["slots"]] = y.view(-1, LATENT)
    rope[st["slots"]] = st["rows"][:, LATENT:ROW].to(F64)
    return {"codes": codes.view(pages, PAGE, LATENT), "rope": rope.view(pages, PAGE, ROPE), "scales": None}


def _exact_rows(st, table):
    """Rows [64 * pages, 576] of one block table in 64 bits, read page by page from the raw bytes."""
    t = table.long()
    if not st["mx8"]:
        return st["cache"][t, 1].to(F64).view(-1, ROW)
    raw = st["cache"][t, 1]
    byte = raw[:, :CODES].long()
    man, exp = byte & 7, (byte >> 3) & 15
    mag = torch.where(exp == 0, man.to(F64) / 8 * 2.0 ** -6, (1 + man.to(F64) / 8) * torch.exp2(exp.to(F64) - 7))
    val = torch.where(byte >= 128, -mag, mag).view(-1, LATENT // 32, 32)
    val = val * torch.exp2(raw[:, SCALES_AT:].to(F64) - 127).reshape(-1, LATENT // 32, 1)
    return torch.cat([val.view(-1, LATENT), raw[:, ROPE_AT:SCALES_AT].contiguous().view(BF16).to(F64).view(-1, ROPE)], 1)


def _exact_attn(st):
    b, s, h = st["batch"], st["steps"], st["heads"]
    shared = _exact_rows(st, st["prefix_table"])[:st["prefix"]]
    lens = st["lens"].tolist()
    out = torch.zeros((b, s, h, LATENT), dtype=F64, device=shared.device)
    for i in range(b):
        mine = _exact_rows(st, st["table"][i][:_pages(lens[i])])
        for j in range(s):
            keys = torch.cat([shared, mine[:max(0, lens[i] - (s - 1 - j))]])
            if keys.shape[0]:
                p = torch.softmax(SOFTMAX_SCALE * (st["q"][i, j].to(F64) @ keys.T), -1)
                out[i, j] = p @ keys[:, :LATENT]
    return out


# ---- what no form can do without ----------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "store":
        return {"bytes": case["tokens"] * (ROW * 2 + 8 + LATENT + LATENT // 32 + ROPE * 2), "flops": 0}
    if case["op"] == "gather":
        return {"bytes": case["tokens"] * (LATENT + LATENT // 32 + ROPE * 2) + case["rows"] * ROW * 2 + 4 * _pages(case["tokens"]), "flops": 0}
    if case["op"] == "verify":
        # one row of the target and one of the draft for each sequence, the drafted tokens' entries, the answers
        b, s, v = case["batch"], case["steps"], case["vocab"]
        return {"bytes": b * (v * 4 * (2 if case["probs"] else 1) + s * (8 + 4 + 4) + 4 + 4 + 8 * (s + 1)), "flops": 0}
    b, s, h = case["batch"], case["steps"], case["heads"]
    lens = _suffix_lens(case)
    row = LATENT + LATENT // 32 + ROPE * 2 if case["mx8"] else ROW * 2
    scores = b * s * h * case["prefix"] + h * sum(max(0, n - (s - 1 - j)) for n in lens for j in range(s))
    return {"bytes": (case["prefix"] + sum(lens)) * row + b * s * h * (ROW + LATENT) * 2, "flops": 2 * (ROW + LATENT) * scores}
