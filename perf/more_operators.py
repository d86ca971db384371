"""The measured cases of the tail of a batched step: what a server needs
between the hidden states of many sequences and their next tokens, beside the
one-row lm_head and argmax.

  product  matrix product in 8-bit integers with a scale for each token and
           each channel, of rows quantized already (mm_int8, int8 rows)
  linear   the same of rows in 16 or 32 bits, quantized within the call
           (mm_int8, floating rows)
  sample   a token for each row of logits: temperature, top-k, top-p and min-p,
           drawn with given random numbers (sample)

  product  y[m, n] = (sum_k x[m, k] w[n, k]) * (xs[m] * ws[n]), the sum in int32
  linear   s = 127 / (max_k |x[m, k]| + 1e-9), q = rint(x s), xs = 1 / s, all in
           binary32; then the product of q
  sample   w_i = exp((l_i - max l) / T).  In the order of falling logits (of
           equal ones the lower index first): the first top_k; of those, the
           ones whose predecessors have less than top_p of the top_k's mass; of
           those, the ones with w_i >= min_p.  The token is the first, in the
           same order, at which the sum of the kept w_i so far exceeds u times
           their whole sum.  T = 0 takes the largest logit.

`own` says which side run() computes: the plain form in elementary torch
operations, or the calls of the framework.  The sizes are those of
BitNet-b1.58-2B (hidden 2560, FFN 6912) and Llama-3.2-1B (hidden 2048, FFN
8192) with their vocabulary of 128256, and generic ones.
"""
import math

import numpy as np
import torch

own = False

VOCAB = 128256


def listed():
    return [
        # one token's projection: the smallest product
        dict(name="linear_token", kind="linear", m=1, k=2560, n=2560, x="float16", out="float16", pad=0),
        # one token's logits, the row quantized by the final norm before
        dict(name="product_token_head", kind="product", m=1, k=2048, n=VOCAB, x="int8", out="float16", pad=0),
        # a small serving batch through a down projection
        dict(name="linear_batch", kind="linear", m=23, k=6912, n=2560, x="bfloat16", out="bfloat16", pad=0),
        # the logits of a serving batch
        dict(name="linear_batch_head", kind="linear", m=96, k=2560, n=VOCAB, x="float16", out="float16", pad=0),
        # odd sizes, rows that are parts of wider ones, the bare integer sums
        dict(name="product_odd_sums", kind="product", m=131, k=997, n=5003, x="int8", out="int32", pad=35),
        # a ragged prefill through an up projection
        dict(name="linear_prefill", kind="linear", m=1021, k=2048, n=8192, x="bfloat16", out="bfloat16", pad=0),
        # a long prefill, the largest
        dict(name="product_prefill_8k", kind="product", m=8192, k=2560, n=6912, x="int8", out="bfloat16", pad=0),
        # one token of one chat
        dict(name="sample_token", kind="sample", m=1, v=VOCAB, x="float16", t=0.8, topk=50, topp=0.95, minp=0.0,
             mixed=False),
        # one token of free text from binary32 logits, nothing cut off, a small vocabulary: the smallest draw
        dict(name="sample_small", kind="sample", m=3, v=32003, x="float32", t=1.0, topk=0, topp=1.0, minp=0.0,
             mixed=False),
        # a serving batch, each sequence with settings of its own
        dict(name="sample_batch", kind="sample", m=64, v=VOCAB, x="bfloat16", t=1.0, topk=200, topp=0.9, minp=0.05,
             mixed=True),
        # a large batch cut by mass alone
        dict(name="sample_large", kind="sample", m=256, v=VOCAB, x="float16", t=1.0, topk=0, topp=0.92, minp=0.0,
             mixed=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: rows from 1 to 8192, any K and N,
    vocabularies of 1000 to 260000."""
    kind = rng.choice(["product", "linear", "sample", "sample"])
    if kind == "sample":
        v = rng.choice([VOCAB, _log_int(rng, 1000, 260000)])
        return dict(kind=kind, m=_log_int(rng, 1, max(1, 256 * VOCAB // (2 * v))), v=v,
                    x=rng.choice(["float16", "bfloat16", "float32"]), t=rng.choice([0.0, 0.3, 0.7, 1.0, 1.7]),
                    topk=rng.choice([0, 0, 1, _log_int(rng, 2, 5000)]),
                    topp=rng.choice([1.0, 1.0, 0.5, rng.uniform(0.7, 0.999)]),
                    minp=rng.choice([0.0, 0.0, rng.uniform(0.001, 0.3)]), mixed=rng.random() < 0.3)
    k = rng.choice([2048, 2560, 6912, 8192, _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)])
    n = rng.choice([512, 640, 2560, 8192, VOCAB if k <= 2560 else 2048, _log_int(rng, 16, 16384)])
    m = rng.choice([_log_int(rng, 1, 16), _log_int(rng, 5, 300), _log_int(rng, 128, 8192)])
    m = max(1, min(m, 8192 * 2560 * 6912 // (k * n), 200000000 // n))
    return dict(kind=kind, m=m, k=k, n=n,
                x="int8" if kind == "product" else rng.choice(["float16", "bfloat16", "float32"]),
                out=rng.choice(["float16", "bfloat16", "float32"] + ["int32"] * (kind == "product")),
                pad=rng.choice([0, 0, 64, 7]))


_BYTES = dict(int8=1, float16=2, bfloat16=2, float32=4, int32=4)


def work(case):
    c = case
    if c["kind"] == "sample":
        # logits read once, settings and u read, token and its probability written; an exponential is about 20
        return dict(bytes=c["m"] * (c["v"] * _BYTES[c["x"]] + 28), flops=25 * c["m"] * c["v"])
    m, k, n = c["m"], c["k"], c["n"]
    scales = 4 * n + (4 * m if c["kind"] == "product" else 0)
    return dict(bytes=n * k + m * k * _BYTES[c["x"]] + m * n * _BYTES[c["out"]] + scales, flops=2 * m * n * k)


def _quantized(x):
    """Rows in 8 bits and their scales."""
    x = x.float()
    s = 127.0 / (x.abs().amax(1) + 1e-9)
    return (x * s[:, None]).round().clamp(-128, 127), 1.0 / s


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    m = c["m"]
    s = dict(case=c)
    if c["kind"] == "sample":
        v = c["v"]
        # most of a vocabulary is unlikely; a few tokens, more in some rows than in others, stand out
        logits = normal(m, v) * 1.8 - 4.0
        few = (uniform(m, 64) * v).long()
        logits.scatter_(1, few, 4.0 - uniform(m, 64) * torch.arange(64, device="cuda") * (0.1 + 0.4 * uniform(m, 1)))
        s["logits"] = logits.to(getattr(torch, c["x"]))
        s["u"] = uniform(m)
        s["t"], s["topk"], s["topp"], s["minp"] = c["t"], c["topk"], c["topp"], c["minp"]
        if c["mixed"]:  # each row its own settings, on the device
            i = torch.arange(m, device="cuda")
            s["t"] = (c["t"] * (0.5 + uniform(m))) * (i % 8 != 3)  # one row in eight takes the largest
            s["topk"] = torch.where(i % 2 == 0, c["topk"], 0) + (uniform(m) * 40).int() * (i % 2 == 0)
            s["topk"] = s["topk"].to(torch.int32)
            s["topp"] = torch.where(i % 3 == 0, c["topp"] * (0.8 + 0.2 * uniform(m)), 1.0)
            s["minp"] = torch.where(i % 5 == 0, c["minp"] * uniform(m), 0.0)
        s["prob"] = torch.empty(m, device="cuda")
        if own:
            import ter_amd
            s["sample"] = ter_amd.sample
        return s
    k, n = c["k"], c["n"]
    # channels of different sizes; activations with a few large channels
    w = normal(n, k) * (0.01 + 0.03 * uniform(n, 1))
    s["w"], s["ws"] = _quantized(w)
    s["w"] = s["w"].to(torch.int8)
    del w
    x = normal(m, k + c["pad"]) * (0.5 + uniform(m, 1))
    x *= 1 + 14 * (uniform(k + c["pad"]) < 0.004)
    if c["kind"] == "product":
        x, s["xs"] = _quantized(x)
    s["x"] = x.to(getattr(torch, c["x"]))[:, :k]
    s["out"] = getattr(torch, c["out"])
    if own:
        import ter_amd
        s["mm"], s["weights"] = ter_amd.mm_int8, ter_amd.PackedInt8.from_int8(s["w"], s["ws"])
    return s


def run(state):
    s = state
    c = s["case"]
    if c["kind"] == "sample":
        if own:
            token = s["sample"](s["logits"], s["u"], temperature=s["t"], top_k=s["topk"], top_p=s["topp"],
                                min_p=s["minp"], prob_out=s["prob"])
            return dict(token=token, prob=s["prob"])
        return _sample(s)
    if own:
        return s["mm"](s["weights"], s["x"], s.get("xs"), dtype=s["out"])
    return _product(s)


def _product(s):
    if s["out"] == torch.int32:  # (sums past 2^24)
        return (s["x"].double() @ s["w"].double().t()).to(torch.int32)
    x, xs = (s["x"].float(), s["xs"]) if "xs" in s else _quantized(s["x"])
    return ((x @ s["w"].float().t()) * (xs[:, None] * s["ws"])).to(s["out"])


def _sample(s):
    """The exponentials and their sums in 64 bits: a token changes where a sum
    crosses u times the whole."""
    x = s["logits"].float()
    m, v = x.shape

    def row(p, dtype):
        return torch.as_tensor(p, device="cuda").to(dtype).expand(m)[:, None]

    t, k = row(s["t"], torch.float32).double(), row(s["topk"], torch.int64)
    # (settings are binary32)
    p, q = (row(s[n], torch.float32).double() for n in ("topp", "minp"))
    k = torch.where(t > 0, torch.where(k > 0, k, v), 1)
    w = ((x - x.amax(1, keepdim=True)).double() / torch.where(t > 0, t, 1.0)).exp()
    order = x.sort(dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order) * (torch.arange(v, device="cuda") < k)
    before = ranked.cumsum(1) - ranked
    keep = (before < p * ranked.sum(1, keepdim=True)) & (ranked >= q) & (torch.arange(v, device="cuda") < k)
    upto = (ranked * keep).cumsum(1)
    total = upto[:, -1:]
    at = (upto <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    token, prob = order.gather(1, at), ranked.gather(1, at) / total
    return dict(token=token[:, 0].to(torch.int32), prob=prob[:, 0].float())


def exact(case, seed):
    """From the definitions, rows and channels at a time."""
    c = case
    s = prepare(c, seed)
    if c["kind"] != "sample":
        x, xs = s["x"], s.get("xs")
        if xs is None:  # the steps of the quantization are binary32's by definition
            x = x.float()
            s127 = torch.full((len(x),), 127.0, device="cuda") / (x.abs().max(1).values + torch.tensor(1e-9, device="cuda"))
            x, xs = torch.round(x * s127[:, None]), torch.ones_like(s127) / s127
        x = x.double()
        parts = [x @ w.double().t().contiguous() for w in s["w"].split(16384)]
        sums = torch.cat(parts, 1)
        return sums.to(torch.int32) if c["out"] == "int32" else sums * xs.double()[:, None] * s["ws"].double()
    m, v = c["m"], c["v"]
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()

    def rows(p):
        p = p.cpu().numpy() if isinstance(p, torch.Tensor) else np.float32(p)
        return np.broadcast_to(p, (m,))

    ts, ks, ps, qs = rows(s["t"]), rows(s["topk"]), rows(s["topp"]), rows(s["minp"])
    token, prob = np.zeros(m, np.int32), np.zeros(m)
    for r in range(m):
        x = logits[r].astype(np.longdouble)  # 64 bits of mantissa
        order = np.argsort(-logits[r], kind="stable")
        if not ts[r] > 0:
            token[r], prob[r] = order[0], 1.0
            continue
        w = np.exp((x - x.max()) / np.longdouble(ts[r]))
        first = order[:int(ks[r])] if 0 < ks[r] < v else order
        mass = np.cumsum(w[first])
        n = 1 + int(np.searchsorted(mass, np.longdouble(ps[r]) * mass[-1]))
        kept = first[:n][w[first[:n]] >= qs[r]]
        sums = np.cumsum(w[kept])
        i = int(np.searchsorted(sums, np.longdouble(u[r]) * sums[-1], side="right"))
        token[r], prob[r] = kept[i], w[kept[i]] / sums[-1]
    return dict(token=torch.from_numpy(token), prob=torch.from_numpy(prob))
