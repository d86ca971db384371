"""The tail of a batched step as a server runs it: hidden states of many
sequences, their logits by the 8-bit head, a token for each; eager and as one
graph, beside the paged attention that makes such hidden states."""
import pytest
import torch

import ter_amd as T
from tests.int8_ref import product, quantized
from tests.sample_ref import draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 3, 20, 70])
def test_from_hidden_states_to_tokens(cuda, m):
    h, v = 640, 9001
    g = torch.Generator().manual_seed(m)
    emb = (torch.randn(v, h, generator=g) * 0.05).half()
    W = T.PackedInt8.quantize(emb.cuda())
    w, ws = quantized(emb)
    i = torch.arange(m)
    kw = dict(temperature=0.7 + 0.6 * torch.rand(m, generator=g), top_k=(40 * (i % 2)).int(),
              top_p=torch.where(i % 3 == 0, 0.9, 1.0), min_p=torch.where(i % 4 == 3, 0.02, 0.0))
    dev = {k: p.cuda() for k, p in kw.items()}
    hidden = torch.empty(m, h, dtype=torch.bfloat16, device="cuda")
    u = torch.empty(m, device="cuda")
    token = torch.empty(m, dtype=torch.int32, device="cuda")

    def step():
        logits = T.mm_int8(W, hidden, dtype=torch.float16)
        return T.sample(logits, u, out=token, **dev)

    def one(seed):
        g = torch.Generator().manual_seed(seed)
        x, r = (torch.randn(m, h, generator=g) * 2).bfloat16(), torch.rand(m, generator=g)
        hidden.copy_(x)
        u.copy_(r)
        logits = product(*quantized(x), w, ws, torch.float16).double().numpy()
        return [draw(logits[b], r[b].item(), **{k: p[b].item() for k, p in kw.items()})[0] for b in range(m)]

    want = one(1)
    assert step().tolist() == want
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (2, 3, 4):
        want = one(seed)
        token.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert token.tolist() == want
        assert step().tolist() == want


def test_behind_the_paged_attention(cuda):
    """A decode step's attention, its output projected in 8 bits, a token for
    each sequence: one graph, replayed over growing contexts."""
    nh, nkv, d, ps, n, v = 8, 2, 64, 16, 5, 5003
    g = torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").half()

    kc, vc = normal(40, ps, nkv, d), normal(40, ps, nkv, d)
    pages = torch.randperm(40, generator=g, device="cuda")[:n * 6].view(n, 6).int()
    lens = torch.tensor([3, 17, 40, 64, 90], dtype=torch.int32, device="cuda")
    attn = T.PagedAttention(nh, nkv, d, 128, 10000.0, neox=True, dtype=torch.float16)
    cache = T.PagedCache(kc, vc)
    batch = T.PagedBatch(torch.arange(n + 1, dtype=torch.int32, device="cuda"), lens, pages)
    head = T.PackedInt8.quantize(normal(v, nh * d))
    q, u = normal(n, nh, d), torch.rand(n, generator=g, device="cuda")

    def step():
        out = attn.attend(q, cache, batch)
        logits = T.mm_int8(head, out.view(n, nh * d), dtype=torch.float32)
        return logits, T.sample(logits, u, temperature=0.8, top_k=50, top_p=0.95)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, token = step()
    for _ in range(3):
        lens += 1
        q.copy_(normal(n, nh, d))
        graph.replay()
        torch.cuda.synchronize()
        again, t = step()
        assert torch.equal(logits, again) and torch.equal(token, t)
        x = logits.double().cpu().numpy()
        assert token.tolist() == [draw(x[b], u[b].item(), 0.8, 50, 0.95)[0] for b in range(n)]


def test_two_tails_at_once(cuda):
    """Two graphs on two streams, each with its own workspaces, beside eager
    calls on a third."""
    h, v = 1030, 20011
    g = torch.Generator(device="cuda").manual_seed(11)
    W = T.PackedInt8.quantize(torch.randn(v, h, generator=g, device="cuda"))
    parts = []
    for m in (70, 20):
        x, u = torch.randn(m, h, generator=g, device="cuda").half(), torch.rand(m, generator=g, device="cuda")

        def step(x=x, u=u):
            return T.sample(T.mm_int8(W, x), u, temperature=0.9, top_p=0.95)

        want = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            token = step()
        parts.append((graph, token, want, step, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, token, _, _, st in parts:
            with torch.cuda.stream(st):
                token.fill_(-2)
                for _ in range(4):
                    graph.replay()
        eager = [step() for _, _, _, step, _ in parts]
        torch.cuda.synchronize()
        for (_, token, want, _, _), e in zip(parts, eager):
            assert torch.equal(token, want) and torch.equal(e, want)
