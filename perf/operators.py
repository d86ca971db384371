"""The measured cases of the paged-cache operators: what a server needs to run
prompts and batches of sequences beside the one-sequence decode attention.

  append   rotary positions of the new queries and keys of a batch of
           sequences, the keys and values written to their cache pages
           (PagedAttention.append)
  attend   causal attention of the new rows of every sequence, prompts and
           single tokens mixed, over its cache pages (PagedAttention.attend)
  shared   the same where all sequences begin with the same pages: the common
           prefix is computed once for all of them (attend(..., shared=n))

With h = query head, g(h) its KV head, row i of a sequence at position p and
angles a_k = p * theta^(-2k/d):
  append   (x_a, x_b) -> (x_a cos a_k - x_b sin a_k, x_a sin a_k + x_b cos a_k),
           (a, b) = (k, k + d/2) or (2k, 2k + 1)
  attend   out[i, h] = sum_{s <= p} softmax_s(q[i, h] . K[s, g(h)] / sqrt(d)) V[s, g(h)]

`own` says which side run() computes: the plain form in elementary torch
operations, or the calls of the framework.  The head shapes are those of
BitNet-b1.58-2B (20 query heads on 5 KV heads of 128) and Llama-3.2-1B (32 on
8 of 64), and generic ones in draw().
"""
import math

import numpy as np
import torch

own = False

THETA = 500000.0
BITNET = dict(nh=20, nkv=5, hd=128, neox=True)
LLAMA = dict(nh=32, nkv=8, hd=64, neox=False)


def listed():
    return [
        # one new token of one sequence early in a chat, one layer
        dict(name="append_token", kind="append", seqs=1, rows="ones", ctx="even", cmax=1500, page=16, dtype="float16",
             **BITNET),
        # a serving batch, one new token each, contexts of every length
        dict(name="append_batch", kind="append", seqs=192, rows="ones", ctx="log", cmax=4000, page=64,
             dtype="bfloat16", **LLAMA),
        # the prompts of a prefill step, 1 to 4000 tokens long
        dict(name="append_prompts", kind="append", seqs=13, rows="log", rmax=4000, ctx="none", cmax=0, page=32,
             dtype="float16", **BITNET),
        # one token of one short chat: the smallest attention
        dict(name="attend_token", kind="attend", seqs=1, rows="ones", ctx="even", cmax=777, page=16, dtype="float16",
             **LLAMA),
        # one token over a long document
        dict(name="attend_long", kind="attend", seqs=1, rows="ones", ctx="even", cmax=65520, page=64,
             dtype="bfloat16", **BITNET),
        # a serving batch of single tokens over contexts of 1 to 4096
        dict(name="attend_batch", kind="attend", seqs=96, rows="ones", ctx="lin", cmax=4095, page=16,
             dtype="float16", **LLAMA),
        # a prefill step: ragged prompts, some behind a cached context
        dict(name="attend_prompts", kind="attend", seqs=9, rows="log", rmax=2900, ctx="some", cmax=1500, page=32,
             dtype="float16", **BITNET),
        # a continuous batch: single tokens beside chunks of new prompts
        dict(name="attend_mixed", kind="attend", seqs=40, rows="chunk", rmax=500, ctx="lin", cmax=3500, page=64,
             dtype="bfloat16", **LLAMA),
        # one long prompt, the largest
        dict(name="attend_prompt_16k", kind="attend", seqs=1, rows="even", rmax=16384, ctx="none", cmax=0, page=64,
             dtype="bfloat16", **BITNET),
        # a few samples of one short prompt, one token each
        dict(name="shared_few", kind="shared", seqs=4, rows="ones", ctx="log", cmax=60, prefix=448, page=16,
             dtype="float16", **BITNET),
        # a large batch behind one system prompt
        dict(name="shared_batch", kind="shared", seqs=128, rows="ones", ctx="log", cmax=500, prefix=8192, page=64,
             dtype="bfloat16", **LLAMA),
        # candidate answers scored behind one long question; the prefix ends inside a page
        dict(name="shared_answers", kind="shared", seqs=24, rows="log", rmax=40, ctx="none", cmax=0, prefix=5991,
             page=32, dtype="float16", **BITNET),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: head shapes of groups 1 to 12, pages
    of 16 to 256 positions, any lengths."""
    kind = rng.choice(["append", "attend", "attend", "shared"])
    heads = rng.choice([BITNET, LLAMA, dict(nh=8, nkv=8, hd=64, neox=True), dict(nh=12, nkv=4, hd=128, neox=False),
                        dict(nh=16, nkv=2, hd=128, neox=True), dict(nh=12, nkv=1, hd=64, neox=True)])
    c = dict(kind=kind, page=rng.choice([16, 32, 48, 64, 128, 256]), dtype=rng.choice(["float16", "bfloat16"]),
             **heads)
    if kind == "append":
        form = rng.choice(["ones", "log", "even"])
        n = _log_int(rng, 1, 256 if form == "ones" else 12)
        return dict(c, seqs=n, rows=form, rmax=_log_int(rng, 1, 4000), ctx=rng.choice(["none", "lin", "log"]),
                    cmax=rng.randrange(1, 4000))
    if kind == "shared":
        n = _log_int(rng, 2, 128)
        r = 1 if rng.random() < 0.6 else _log_int(rng, 1, max(1, 512 // n))
        return dict(c, seqs=n, rows="ones" if r == 1 else "log", rmax=r, ctx=rng.choice(["none", "log"]),
                    cmax=_log_int(rng, 1, 500), prefix=_log_int(rng, 100, 8192))
    form = rng.choice(["token", "batch", "prompts", "chunk"])
    if form == "token":
        return dict(c, seqs=_log_int(rng, 1, 4), rows="ones", ctx="even", cmax=_log_int(rng, 1, 65000))
    if form == "batch":
        return dict(c, seqs=_log_int(rng, 2, 128), rows="ones", ctx=rng.choice(["lin", "log"]),
                    cmax=_log_int(rng, 30, 4000))
    if form == "prompts":
        n = _log_int(rng, 1, 10)
        return dict(c, seqs=n, rows="log", rmax=_log_int(rng, 20, 8000 // n + 200), ctx=rng.choice(["none", "some"]),
                    cmax=rng.randrange(1, 2000))
    return dict(c, seqs=_log_int(rng, 2, 48), rows="chunk", rmax=_log_int(rng, 2, 400), ctx="lin",
                cmax=rng.randrange(100, 3500))


def _lengths(c):
    """(new rows, cached positions behind the prefix) of every sequence: by
    the case alone, so that work() knows them too."""
    n = c["seqs"]
    r = np.random.RandomState(n * 7919 + c["cmax"] * 31 + c.get("rmax", 1))
    rmax, cmax = c.get("rmax", 1), c["cmax"]
    if c["rows"] == "ones":
        rows = np.ones(n, np.int64)
    elif c["rows"] == "even":
        rows = np.full(n, rmax, np.int64)
    elif c["rows"] == "log":
        rows = np.exp(r.uniform(0, math.log(rmax + 0.5), n)).round().astype(np.int64).clip(1, rmax)
        rows[0] = rmax
    else:  # "chunk": one sequence in eight is a piece of a prompt
        rows = np.where(np.arange(n) % 8 == 1, r.randint(max(1, rmax // 2), rmax + 1, n), 1)
    if c["ctx"] == "none":
        ctx = np.zeros(n, np.int64)
    elif c["ctx"] == "even":
        ctx = np.full(n, cmax, np.int64)
    elif c["ctx"] == "lin":
        ctx = r.randint(0, cmax + 1, n)
    elif c["ctx"] == "log":
        ctx = np.exp(r.uniform(0, math.log(cmax + 0.5), n)).round().astype(np.int64)
    else:  # "some": every other sequence has a context
        ctx = np.where(np.arange(n) % 2 == 1, r.randint(0, cmax + 1, n), 0)
    return rows.astype(np.int64), ctx.astype(np.int64)


def work(case):
    c = case
    rows, ctx = _lengths(c)
    nh, nkv, d, pre = c["nh"], c["nkv"], c["hd"], c.get("prefix", 0)
    t = int(rows.sum())
    if c["kind"] == "append":
        # q, k and v read once; rotated q, cached k and v written once; 3 operations an element rotated
        return dict(bytes=2 * 2 * t * (nh + 2 * nkv) * d, flops=3 * t * (nh + nkv) * d)
    # q read and out written; every visible position's key and value read once (the prefix once for all)
    kv = int((rows + ctx).sum()) + pre
    pairs = int((rows * (pre + ctx) + rows * (rows + 1) // 2).sum())
    return dict(bytes=2 * (2 * t * nh * d + 2 * kv * nkv * d), flops=4 * pairs * nh * d)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = getattr(torch, c["dtype"])
    nh, nkv, d, ps, n = c["nh"], c["nkv"], c["hd"], c["page"], c["seqs"]
    rows, ctx = _lengths(c)
    pre = c.get("prefix", 0)
    lens = pre + ctx + rows
    need = -(-lens // ps)
    common = pre // ps  # whole pages of the prefix, the same for all; a page that the prefix ends in is each one's own copy
    width = int(need.max())
    n_pages = int((need - common).sum()) + common + 3
    # pages in the order that an allocator hands them out after a while: any
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    at = np.full((n, width), -1, np.int64)
    at[:, :common] = np.arange(common)
    nxt = common
    for b in range(n):
        k = int(need[b]) - common
        at[b, common:common + k] = np.arange(nxt, nxt + k)
        nxt += k
    at = torch.from_numpy(at).cuda()
    pages = torch.where(at >= 0, ids[at.clamp(min=0)], torch.full_like(at, -1, dtype=torch.int32))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    # keys of a trained model have a few channels with a large mean; queries answer to them
    mean = normal(nkv, d) * (torch.rand(nkv, d, generator=g, device="cuda") < 0.06) * 3
    kc = torch.empty(n_pages, ps, nkv, d, dtype=dt, device="cuda")
    vc = torch.empty_like(kc)
    for p in range(0, n_pages, 4096):  # (in pieces: the fp32 draws of a large cache)
        m = min(4096, n_pages - p)
        kc[p:p + m] = (normal(m, ps, nkv, d) + mean).to(dt)
        vc[p:p + m] = normal(m, ps, nkv, d).to(dt)
    if common < -(-pre // ps):
        # the last, partly filled page of the prefix: the same contents in every sequence's copy
        copies = pages[:, common].long()
        kc[copies, :pre % ps] = kc[copies[0], :pre % ps].clone()
        vc[copies, :pre % ps] = vc[copies[0], :pre % ps].clone()
    t = int(rows.sum())
    first = np.concatenate([[0], np.cumsum(rows)])
    s = dict(case=c, q=(normal(t, nh, d) * 1.2).to(dt), kc=kc, vc=vc, pages=pages,
             rows=torch.tensor(first, dtype=torch.int32, device="cuda"),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             most=int(rows.max()), longest=int(lens.max()), shared=common * ps)
    if c["kind"] == "append":
        s["k"] = (normal(t, nkv, d) + mean).to(dt)
        s["v"] = normal(t, nkv, d).to(dt)
    if own:
        import ter_amd as T
        s["attn"] = T.PagedAttention(nh, nkv, d, s["longest"], THETA, neox=c["neox"], dtype=dt)
        s["cache"] = T.PagedCache(kc, vc)
        s["batch"] = T.PagedBatch(s["rows"], s["lens"], pages)
    return s


def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        if kind == "append":
            q = s["attn"].append(s["q"], s["k"], s["v"], s["cache"], s["batch"])
            return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])
        return s["attn"].attend(s["q"], s["cache"], s["batch"], shared=s["shared"] if kind == "shared" else 0)
    if kind == "append":
        return _append(s)
    return _attend(s, s["shared"] if kind == "shared" else 0)


def _places(s):
    """Sequence and position of every new row."""
    t = s["q"].shape[0]
    i = torch.arange(t, device="cuda")
    first = s["rows"].long()
    b = torch.searchsorted(first, i, right=True) - 1
    return b, s["lens"].long()[b] - first[b + 1] + i


def _append(s):
    c = s["case"]
    b, pos = _places(s)
    d = c["hd"]
    # angles of far positions in 64 bits
    ang = pos.double()[:, None] * THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def rotate(x):
        x = x.float()
        if c["neox"]:
            u, v = x[..., :d // 2], x[..., d // 2:]
            return torch.cat([u * cos - v * sin, u * sin + v * cos], -1).to(s["q"].dtype)
        u, v = x[..., 0::2], x[..., 1::2]
        return torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2).to(s["q"].dtype)

    page, slot = s["pages"].long()[b, pos // c["page"]], pos % c["page"]
    s["kc"][page, slot] = rotate(s["k"])
    s["vc"][page, slot] = s["v"]
    return dict(q=rotate(s["q"]), k_cache=s["kc"], v_cache=s["vc"])


def _attend(s, shared):
    """All sequences padded to the longest, in 32 bits; the shared prefix is
    gathered and multiplied once."""
    c = s["case"]
    nkv, d, ps, n, r = c["nkv"], c["hd"], c["page"], c["seqs"], s["most"]
    grp = c["nh"] // nkv
    b, pos = _places(s)
    at = torch.arange(s["q"].shape[0], device="cuda") - s["rows"].long()[b]  # row within its sequence
    q = torch.zeros(n, r, nkv, grp, d, device="cuda")
    q[b, at] = s["q"].float().view(-1, nkv, grp, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, nkv, r * grp, d)
    where = torch.full((n, r), -1, device="cuda")
    where[b, at] = pos
    where = where.repeat_interleave(grp, 1)[:, None, :, None]  # position of each row

    def gather(cache, table, positions):
        x = cache[table.long().clamp(min=0)[:, positions // ps], positions % ps].float()
        return x.permute(0, 2, 1, 3).contiguous()  # [n, nkv, positions, d]

    own_at = torch.arange(shared, s["longest"], device="cuda")
    score = torch.matmul(q, gather(s["kc"], s["pages"], own_at).transpose(2, 3).contiguous())
    score.mul_(d ** -0.5).masked_fill_(own_at > where, -math.inf)
    if shared:
        pre_at = torch.arange(shared, device="cuda")
        k = gather(s["kc"], s["pages"][:1], pre_at)[0]
        flat = q.transpose(0, 1).reshape(nkv, n * r * grp, d)
        pre = torch.matmul(flat, k.transpose(1, 2).contiguous()).view(nkv, n, r * grp, shared).transpose(0, 1)
        pre = (pre * d ** -0.5).masked_fill_(pre_at > where, -math.inf)
        score = torch.cat([pre, score], -1)
    score.masked_fill_(where < 0, 0.0)  # padding rows see anything
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score[..., shared:], gather(s["vc"], s["pages"], own_at))
    if shared:
        v = gather(s["vc"], s["pages"][:1], pre_at)[0]
        part = torch.matmul(score[..., :shared].transpose(0, 1).reshape(nkv, n * r * grp, shared), v)
        out += part.view(nkv, n, r * grp, d).transpose(0, 1)
    out /= total
    out = out.view(n, nkv, r, grp, d).permute(0, 2, 1, 3, 4)[b, at]
    return out.reshape(-1, c["nh"], d).to(s["q"].dtype)


def exact(case, seed):
    """From the definitions, one sequence and KV head at a time, in 64 bits."""
    c = case
    s = prepare(c, seed)
    rows, ctx = _lengths(c)
    nh, nkv, d, ps = c["nh"], c["nkv"], c["hd"], c["page"]
    grp = nh // nkv
    first = np.concatenate([[0], np.cumsum(rows)])
    lens = rows + ctx + c.get("prefix", 0)
    if c["kind"] == "append":
        k, v, q = s["kc"].double(), s["vc"].double(), torch.empty_like(s["q"], dtype=torch.float64)
        freq = torch.tensor([THETA ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device="cuda")
        a, z = ((slice(0, d // 2), slice(d // 2, d)) if c["neox"] else (slice(0, d, 2), slice(1, d, 2)))
        for b in range(c["seqs"]):
            i, j = int(first[b]), int(first[b + 1])
            p = torch.arange(int(lens[b] - rows[b]), int(lens[b]), device="cuda")
            turn = torch.polar(torch.ones(len(p), d // 2, dtype=torch.float64, device="cuda"), p[:, None] * freq)

            def turned(x):
                x = x.double()
                w = torch.complex(x[..., a], x[..., z]) * turn[:, None]
                y = torch.empty_like(x)
                y[..., a], y[..., z] = w.real, w.imag
                return y

            q[i:j] = turned(s["q"][i:j])
            page = s["pages"][b].long()[p // ps]
            k[page, p % ps] = turned(s["k"][i:j])
            v[page, p % ps] = s["v"][i:j].double()
        return dict(q=q, k_cache=k, v_cache=v)
    out = torch.empty_like(s["q"], dtype=torch.float64)
    for b in range(c["seqs"]):
        i, j, m = int(first[b]), int(first[b + 1]), int(lens[b])
        p = torch.arange(m, device="cuda")
        page = s["pages"][b].long()[p // ps]
        hidden = p[None] > torch.arange(m - (j - i), m, device="cuda")[:, None]
        for h in range(nkv):
            k, v = s["kc"][page, p % ps, h].double(), s["vc"][page, p % ps, h].double()
            for e in range(h * grp, h * grp + grp):
                w = (s["q"][i:j, e].double() @ k.T) / math.sqrt(d)
                out[i:j, e] = torch.softmax(w.masked_fill_(hidden, -math.inf), -1) @ v
    return out
