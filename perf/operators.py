"""Measured cases of the paged serving operators (mimo_moe.paged): the page plan of a step, the RoPE + append into a
paged KV cache, and the attention of new tokens over it.

A step of a serving loop has R requests.  Request r holds lens[r] tokens in pages of a pool and brings new[r] new
ones; the step's token rows are the requests' new tokens one request after another, padded to a fixed row count.

  plan  pages for the new tokens from the free list, the row offsets, each row's position and cache slot
  rope  the q | k | v projection rows: RoPE at each row's position, k and v into their slots
  attn  softmax attention of each new token over its request's pages (causal, optionally a sliding window with a
        few first tokens that stay visible, optionally a sink logit per head)

`own` false: elementary torch operations.  `own` true: the calls a user makes."""
import math
import random

import numpy as np
import torch

own = False

# Attention shapes: the full-attention and sliding-window layers of this repository's default configuration, and the
# two other head layouts its attention tests use.
KINDS = {
    "full": dict(n_heads=64, n_kv_heads=4, head_dim=192, v_head_dim=128, rotary_dim=64, rope_theta=5_000_000.0,
                 window=0, sinks=False),
    "swa": dict(n_heads=64, n_kv_heads=8, head_dim=192, v_head_dim=128, rotary_dim=64, rope_theta=10_000.0,
                window=128, sinks=True),
    "d128": dict(n_heads=64, n_kv_heads=8, head_dim=128, v_head_dim=128, rotary_dim=128, rope_theta=5_000_000.0,
                 window=0, sinks=False),
    "d64": dict(n_heads=8, n_kv_heads=8, head_dim=64, v_head_dim=64, rotary_dim=32, rope_theta=5_000_000.0,
                window=0, sinks=False),
}
V_SCALE = 0.70703125   # a value scale that is a bf16 number
PAGES = (16, 32, 64, 128)


def listed():
    return [
        # the bookkeeping of one decode step: the smallest call of a serving loop, 8 requests of a 4096-token context
        dict(name="plan decode 8", op="plan", decodes=8, chunks=0, chunk=0, ctx=4096, ragged=False, page=64, pad=0,
             shape=1),
        # a busy step with chunked prefill: 200 decoding requests and 3 prompts' chunks, rows padded for a graph
        dict(name="plan mixed 203", op="plan", decodes=200, chunks=3, chunk=2048, ctx=32768, ragged=True, page=16,
             pad=77, shape=2),
        # many prompts admitted at once: 1024 requests' first chunks of at most 128 tokens
        dict(name="plan prompts 1024", op="plan", decodes=0, chunks=1024, chunk=128, ctx=0, ragged=True, page=16,
             pad=0, shape=3),
        # one decode step's projection rows of a full-attention layer
        dict(name="rope decode 8", op="rope", kind="full", decodes=8, chunks=0, chunk=0, ctx=4096, ragged=False,
             page=64, pad=0, shape=4),
        # a 2048-token prefill chunk of a full-attention layer
        dict(name="rope chunk 2048", op="rope", kind="full", decodes=0, chunks=1, chunk=2048, ctx=0, ragged=False,
             page=64, pad=0, shape=5),
        # some 16000 prompt tokens of several requests on a sliding-window layer (value scale on), ragged, padded rows
        dict(name="rope ragged prompts", op="rope", kind="swa", decodes=5, chunks=7, chunk=2900, ctx=2000, ragged=True,
             page=16, pad=301, shape=6),
        # decode of 8 requests at a 4096-token context, full attention
        dict(name="attn decode 8", op="attn", kind="full", decodes=8, chunks=0, chunk=0, ctx=4096, ragged=False,
             page=64, pad=0, keep=0, shape=7),
        # decode of 64 requests whose contexts run from a few tokens to 32768, small pages
        dict(name="attn decode ragged 64", op="attn", kind="full", decodes=64, chunks=0, chunk=0, ctx=32768,
             ragged=True, page=16, pad=0, keep=0, shape=8),
        # decode of 48 requests on a sliding-window layer with sink logits and 4 first tokens that stay visible
        dict(name="attn decode window 48", op="attn", kind="swa", decodes=48, chunks=0, chunk=0, ctx=16384,
             ragged=True, page=16, pad=0, keep=4, shape=9),
        # a 2048-token prompt from an empty cache, full attention
        dict(name="attn chunk 2048", op="attn", kind="full", decodes=0, chunks=1, chunk=2048, ctx=0, ragged=False,
             page=64, pad=0, keep=0, shape=10),
        # a step that mixes 23 decoding requests with two prompts' chunks, heads of 128, rows padded
        dict(name="attn mixed d128", op="attn", kind="d128", decodes=23, chunks=2, chunk=1024, ctx=8192, ragged=True,
             page=32, pad=19, keep=0, shape=11),
        # the last 4096-token chunk of a 16384-token prompt, full attention: the largest call
        dict(name="attn chunk 4096 of 16384", op="attn", kind="full", decodes=0, chunks=1, chunk=4096, ctx=12288,
             ragged=False, page=128, pad=0, keep=0, shape=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attn", "attn"])
    page = rng.choice(PAGES)
    c = dict(op=op, page=page, pad=rng.choice([0, 0, rng.randint(1, 200)]), ragged=rng.random() < 0.7,
             shape=rng.randrange(1 << 30))
    form = rng.choice(["decode", "chunk", "mixed"])
    if op == "plan":
        c["decodes"] = _log_int(rng, 1, 1024) if form != "chunk" else 0
        c["chunks"] = _log_int(rng, 1, 32) if form != "decode" else 0
        c["chunk"] = _log_int(rng, 2, 4096) if form != "decode" else 0
        c["ctx"] = _log_int(rng, 1, 32768)
        return c
    if op == "rope":
        c["kind"] = rng.choice(sorted(KINDS))
        c["decodes"] = _log_int(rng, 1, 256) if form != "chunk" else 0
        c["chunks"] = rng.randint(1, 4) if form != "decode" else 0
        c["chunk"] = _log_int(rng, 2, 3500) if form != "decode" else 0
        c["ctx"] = _log_int(rng, 1, 4096)
        return c
    c["kind"] = rng.choice(sorted(KINDS))
    c["decodes"] = _log_int(rng, 1, 64) if form != "chunk" else 0
    c["chunks"] = rng.randint(1, 3) if form != "decode" else 0
    c["chunk"] = _log_int(rng, 2, 4096 // c["chunks"]) if form != "decode" else 0
    c["ctx"] = _log_int(rng, 1, 32768 if form == "decode" else 12288)
    c["keep"] = rng.choice([0, 4, rng.randint(1, 300)]) if KINDS[c["kind"]]["window"] else 0
    return c


def _lengths(case):
    """Tokens each request holds before the step and the new ones it brings (the same for every seed)."""
    rng = random.Random(case["shape"])
    held, new = [], []
    for i in range(case["decodes"] + case["chunks"]):
        if not case["ragged"]:
            held.append(case["ctx"])
        else:
            held.append(_log_int(rng, 1, case["ctx"] + 1) - 1)
        if i < case["decodes"]:
            new.append(1)
        else:
            new.append(rng.randint(max(1, case["chunk"] // 2), case["chunk"]) if case["ragged"] else case["chunk"])
    return held, new


def work(case):
    held, new = _lengths(case)
    rows, P = sum(new), case["page"]
    if case["op"] == "plan":
        R, T = len(new), rows + case["pad"]
        fresh = sum((h + n + P - 1) // P - (h + P - 1) // P for h, n in zip(held, new))
        old = sum(1 for h in held if h % P)            # partly filled pages the new tokens continue in
        # lens, new lens, the touched table entries and free pages read; offsets, lens, table entries, positions, slots
        return {"bytes": 8 * R + 4 * old + 4 * fresh + 4 * (2 * R + 2) + 4 * fresh + 8 * T, "flops": 0}
    k = KINDS[case["kind"]]
    nq, nkv, d, dv = k["n_heads"], k["n_kv_heads"], k["head_dim"], k["v_head_dim"]
    if case["op"] == "rope":
        width = nq * d + nkv * (d + dv)
        return {"bytes": rows * (4 * width + 8), "flops": rows * (nq + nkv) * k["rotary_dim"] * 3}
    pairs = keys = 0
    for h, n in zip(held, new):
        w, keep = k["window"], case["keep"]
        pos = np.arange(h, h + n, dtype=np.int64)
        seen = pos + 1
        first = 0
        if w:
            lo = np.maximum(pos - w + 1, 0)
            seen = pos - lo + 1 + np.minimum(lo, keep)
            first = int(lo[0])
        pairs += int(seen.sum())
        keys += h + n - first + min(first, keep if w else 0)
    return {"bytes": 2 * (keys * nkv * (d + dv) + rows * nq * (d + dv)), "flops": 2 * pairs * nq * (d + dv)}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    held, new = _lengths(case)
    R, P, rows = len(new), case["page"], sum(new)
    T = rows + case["pad"]
    before = [-(-h // P) for h in held]
    after = [-(-(h + n) // P) for h, n in zip(held, new)]
    total = sum(after)
    num_pages = total + 3 + total // 16
    perm = torch.randperm(num_pages, generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    owned = before if case["op"] == "plan" else after
    width = max(after) + 1
    own_n = torch.tensor(owned, device=dev)
    first = torch.cumsum(own_n, 0) - own_n
    col = torch.arange(width, device=dev)
    table = torch.where(col[None, :] < own_n[:, None],
                        perm[(first[:, None] + col[None, :]).clamp_(max=num_pages - 1)], -1).to(torch.int32)
    held_t = torch.tensor(held, dtype=torch.int32, device=dev)
    new_t = torch.tensor(new, dtype=torch.int32, device=dev)
    s = dict(case=case, held=held, new=new, rows=rows, tokens=T, table=table, page=P, num_pages=num_pages)
    if case["op"] == "plan":
        used = sum(before)
        free = torch.zeros(num_pages, dtype=torch.int32, device=dev)
        free[:num_pages - used] = perm[used:]
        s.update(lens=held_t, new_lens=new_t, free=free,
                 n_free=torch.full((1,), num_pages - used, dtype=torch.int32, device=dev))
        if own:
            from mimo_moe import paged
            s["step"] = paged.PageStep.empty(R, T, table, P)
        return s
    k = KINDS[case["kind"]]
    nq, nkv, d, dv = k["n_heads"], k["n_kv_heads"], k["head_dim"], k["v_head_dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.bfloat16)

    cu = torch.zeros(R + 1, dtype=torch.int32, device=dev)
    cu[1:] = torch.cumsum(new_t, 0)
    seq_lens = held_t + new_t
    row = torch.arange(T, device=dev, dtype=torch.int32)
    req = torch.searchsorted(cu[1:], row, right=True).clamp_(max=R - 1)
    live = row < rows
    pos = torch.where(live, held_t[req] + row - cu[req], -1).to(torch.int32)
    slots = torch.where(live, table[req, (pos // P).clamp_(min=0).long()] * P + pos % P, -1).to(torch.int32)
    s.update(cu=cu, seq_lens=seq_lens, positions=pos, slots=slots,
             k=normal(num_pages, nkv, P, d), v=normal(num_pages, nkv, P, dv))
    if case["op"] == "rope":
        s["qkv"] = normal(T, nq * d + nkv * (d + dv))
        s["q"] = torch.zeros(T, nq, d, dtype=torch.bfloat16, device=dev)
    else:
        s["q"] = normal(T, nq, d)
        s["sinks"] = torch.randn(nq, generator=g, device=dev) if k["sinks"] else None
        s["out"] = torch.zeros(T, nq, dv, dtype=torch.bfloat16, device=dev)
    if own:
        from mimo_moe import paged
        from mimo_moe.layer import AttentionConfig
        keep = case["keep"] if case["op"] == "attn" else 0
        s["cfg"] = AttentionConfig(**k, v_scale=V_SCALE if case["op"] == "rope" and k["window"] else None,
                                   keep_first=keep)
        s["cache"] = paged.PagedKVCache(s["cfg"], num_pages, P, k=s["k"], v=s["v"])
        s["step"] = paged.PageStep(block_table=table, page_size=P, cu_q=cu, seq_lens=seq_lens, positions=pos,
                                   slots=slots)
        if case["op"] == "attn":
            s["plan"] = paged.attention_plan(s["step"], s["cfg"])   # one a step, for all layers of a kind
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        from mimo_moe import paged
        if op == "plan":
            p = paged.page_plan(s["lens"], s["new_lens"], s["table"], s["free"], s["n_free"], s["page"], s["tokens"],
                                out=s["step"])
            return [p.cu_q, p.positions, p.slots, p.seq_lens, p.n_free, s["table"]]
        if op == "rope":
            q = paged.rope_store_paged(s["qkv"], s["cfg"], s["cache"], s["step"], q_out=s["q"])
            return [q, s["k"], s["v"]]
        return [paged.attention_paged(s["q"], s["cache"], s["cfg"], s["step"], s["sinks"], plan=s["plan"],
                                      out=s["out"])]
    return {"plan": _plan, "rope": _rope, "attn": _attn}[op](s)


def _plan(s):
    lens, new, P, table = s["lens"], s["new_lens"], s["page"], s["table"]
    R, T, dev = lens.shape[0], s["tokens"], lens.device
    seq_lens = lens + new
    old = (lens + P - 1) // P
    need = (seq_lens + P - 1) // P - old
    ends = torch.cumsum(need, 0, dtype=torch.int32)
    fresh = torch.arange(table.shape[1], device=dev, dtype=torch.int32)[None, :] - old[:, None]
    at = s["n_free"] - 1 - ((ends - need)[:, None] + fresh)
    table = torch.where((fresh >= 0) & (fresh < need[:, None]), s["free"][at.clamp_(0, s["free"].shape[0] - 1)], table)
    cu = torch.zeros(R + 1, dtype=torch.int32, device=dev)
    cu[1:] = torch.cumsum(new, 0, dtype=torch.int32)
    row = torch.arange(T, device=dev, dtype=torch.int32)
    req = torch.searchsorted(cu[1:], row, right=True).clamp_(max=R - 1)
    live = row < cu[R]
    pos = lens[req] + row - cu[req]
    slots = table[req, (pos // P).clamp_(0, table.shape[1] - 1)] * P + pos % P
    return [cu, torch.where(live, pos, -1), torch.where(live, slots, -1), seq_lens, s["n_free"] - ends[-1:], table]


def _rope(s):
    k = KINDS[s["case"]["kind"]]
    nq, nkv, d, dv, rot = k["n_heads"], k["n_kv_heads"], k["head_dim"], k["v_head_dim"], k["rotary_dim"]
    n, P, half = s["rows"], s["page"], rot // 2
    x = s["qkv"][:n]
    freq = k["rope_theta"] ** (-torch.arange(half, device=x.device, dtype=torch.float64) * 2 / rot)
    ang = s["positions"][:n].double()[:, None] * freq[None, :]
    cos, sin = ang.cos().float()[:, None, :], ang.sin().float()[:, None, :]
    qk = x[:, :(nq + nkv) * d].view(n, nq + nkv, d).float()
    a, b = qk[..., :half], qk[..., half:rot]
    qk = torch.cat([a * cos - b * sin, a * sin + b * cos, qk[..., rot:]], -1).to(torch.bfloat16)
    v = x[:, (nq + nkv) * d:].view(n, nkv, dv)
    if k["window"]:
        v = (v.float() * V_SCALE).to(torch.bfloat16)
    slot = s["slots"][:n].long()
    s["q"][:n] = qk[:, :nq]
    s["k"][slot // P, :, slot % P] = qk[:, nq:]
    s["v"][slot // P, :, slot % P] = v
    return [s["q"], s["k"], s["v"]]


def _attn(s):
    # the decoding requests are one padded batch; a prompt's chunk has a length of its own, so each is another
    out, D = s["out"], s["case"]["decodes"]
    groups = [(0, D)] * (D > 0) + [(r, r + 1) for r in range(D, len(s["new"]))]
    for r0, r1 in groups:
        row0, n = sum(s["new"][:r0]), s["new"][r0]
        row1 = row0 + n * (r1 - r0)
        out[row0:row1] = _attend(s, r0, r1, s["q"][row0:row1].unflatten(0, (r1 - r0, n))).flatten(0, 1)
    return [out]


def _attend(s, r0, r1, q):
    k = KINDS[s["case"]["kind"]]
    nkv, d, w, keep, P = k["n_kv_heads"], k["head_dim"], k["window"], s["case"]["keep"], s["page"]
    B, n, nq, _ = q.shape
    L = max(h + m for h, m in zip(s["held"][r0:r1], s["new"][r0:r1]))
    pages = s["table"][r0:r1, :-(-L // P)].clamp(min=0).long()
    K = s["k"][pages].transpose(1, 2).flatten(2, 3)[:, :, :L].float()          # [B, nkv, L, d]
    V = s["v"][pages].transpose(1, 2).flatten(2, 3)[:, :, :L].float()
    x = q.float().view(B, n, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4)         # [B, nkv, G, n, d]
    at = s["seq_lens"][r0:r1, None] - n + torch.arange(n, device=q.device)[None, :]
    key = torch.arange(L, device=q.device)
    seen = key <= at[..., None]
    if w:
        seen &= (key > at[..., None] - w) | (key < keep)
    score = (x.flatten(2, 3) @ K.transpose(2, 3)).view(B, nkv, nq // nkv, n, L).mul_(d ** -0.5)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if k["sinks"]:
        sink = s["sinks"].view(1, nkv, nq // nkv, 1, 1)
        top = torch.maximum(top, sink)
    p = score.sub_(top).exp_()
    den = p.sum(-1, keepdim=True)
    if k["sinks"]:
        den = den + (sink - top).exp()
    o = (p.flatten(2, 3) @ V).unflatten(2, (nq // nkv, n)) / den
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, nq, -1).to(torch.bfloat16)


def exact(case, seed):
    s = prepare(case, seed)
    held, new, P = s["held"], s["new"], s["page"]
    if case["op"] == "plan":
        table, free, top = s["table"].tolist(), s["free"].tolist(), int(s["n_free"])
        cu, pos, slots = [0], [], []
        for r, (h, n) in enumerate(zip(held, new)):
            for p in range(h, h + n):
                if p % P == 0:                     # the token that opens a page takes the last free one
                    top -= 1
                    table[r][p // P] = free[top]
                pos.append(p)
                slots.append(table[r][p // P] * P + p % P)
            cu.append(cu[-1] + n)
        tail = [-1] * case["pad"]
        lens = [h + n for h, n in zip(held, new)]
        return [torch.tensor(x, dtype=torch.int32) for x in (cu, pos + tail, slots + tail, lens, [top], table)]
    k = KINDS[case["kind"]]
    nq, nkv, d, dv = k["n_heads"], k["n_kv_heads"], k["head_dim"], k["v_head_dim"]
    where = [(r, h + i) for r, (h, n) in enumerate(zip(held, new)) for i in range(n)]
    if case["op"] == "rope":
        x = s["qkv"].double()
        pos = torch.tensor([p for _, p in where], dtype=torch.float64, device=x.device)
        q, kp, vp = s["q"].double(), s["k"].double(), s["v"].double()
        page = s["table"][[r for r, _ in where], [p // P for _, p in where]].long()
        off = torch.tensor([p % P for _, p in where], device=x.device)
        rot, n = k["rotary_dim"], len(where)
        for hd in range(nq + nkv):
            y = x[:n, hd * d:(hd + 1) * d].clone()
            for i in range(rot // 2):
                t = pos * math.exp(-2 * i / rot * math.log(k["rope_theta"]))
                a, b = x[:n, hd * d + i], x[:n, hd * d + i + rot // 2]
                y[:, i] = a * torch.cos(t) - b * torch.sin(t)
                y[:, i + rot // 2] = a * torch.sin(t) + b * torch.cos(t)
            if hd < nq:
                q[:n, hd] = y
            else:
                kp[page, hd - nq, off] = y
        for hk in range(nkv):
            at = (nq + nkv) * d + hk * dv
            vp[page, hk, off] = x[:n, at:at + dv] * (V_SCALE if k["window"] else 1.0)
        return [q, kp, vp]
    out = torch.zeros(s["tokens"], nq, dv, dtype=torch.float64, device=s["q"].device)
    row = 0
    for r, (h, n) in enumerate(zip(held, new)):
        L = h + n
        pages = s["table"][r, :-(-L // P)].long()
        i = torch.arange(h, L, device=out.device)[:, None]
        j = torch.arange(L, device=out.device)[None, :]
        hidden = j > i
        if k["window"]:
            hidden |= (j <= i - k["window"]) & (j >= case["keep"])
        for hk in range(nkv):
            K = s["k"][pages, hk].reshape(-1, d)[:L].double()
            V = s["v"][pages, hk].reshape(-1, dv)[:L].double()
            for hq in range(hk * nq // nkv, (hk + 1) * nq // nkv):
                a = s["q"][row:row + n, hq].double() @ K.t() / math.sqrt(d)
                a[hidden] = -math.inf
                if k["sinks"]:
                    a = torch.cat([a, s["sinks"][hq].double().expand(n, 1)], 1)
                out[row:row + n, hq] = torch.softmax(a, 1)[:, :L] @ V
        row += n
    return [out]
