"""Prompts, a token of each request, then a search: the logits a search starts from are those of the last token its slots have read."""
import pytest
import torch

from tests.test_gpu_decode import DEV, close, cu_of, one_at_a_time, plain_search, stack

pytestmark = pytest.mark.gpu


def test_search_after_a_token():
    import mamba_b200
    s, V, G, K, steps = stack(2, 32, 6), 40, 3, 3, 5
    g = torch.Generator().manual_seed(7)
    embed, weight = torch.randn(V, 32, generator=g).to(DEV), (0.7 * torch.randn(32, V, generator=g)).to(DEV)
    embedding, head = lambda t: embed[t], lambda h: h @ weight
    texts = [torch.randint(0, V, (n,), generator=g).to(DEV) for n in (9, 1, 6)]
    pool = mamba_b200.StatePool(s, G * K + 2)
    for t in pool.pools():
        t.normal_()                                         # (slots that nobody has used hold anything)
    beam_slots = torch.randperm(G * K + 2, generator=g)[: G * K].view(G, K).to(DEV)
    slots, cu_seqlens = beam_slots[:, 0], cu_of([9, 1, 6])
    h = pool.prompts(embedding(torch.cat(texts)), cu_seqlens, slots)
    logits = head(h[cu_seqlens[1:] - 1])
    with torch.no_grad():
        want = torch.stack([head(one_at_a_time(s, embedding(t))[-1]) for t in texts])
    close(logits, want)
    chosen = logits.argmax(-1)
    logits = head(pool.step(embedding(chosen), slots))
    # a call in which a request has nothing new leaves its slot as it is
    before = [t[slots[1]].clone() for t in pool.pools()]
    pool.prompts(torch.zeros(0, 32, device=DEV), cu_of([0]), slots[1:2], resume=torch.tensor([False], device=DEV))
    assert all(torch.equal(a, t[slots[1]]) for a, t in zip(before, pool.pools()))
    tokens, scores = mamba_b200.beam_search(pool, embedding, head, logits, beam_slots, steps, end_token=0)
    prompts = [embedding(torch.cat([t, c[None]])) for t, c in zip(texts, chosen)]
    for r, beams in enumerate(plain_search(s, embed, weight, prompts, K, steps, 0)):
        assert tokens[r].tolist() == [b[0] for b in beams]
        assert torch.allclose(scores[r].double().cpu(), torch.tensor([b[1] for b in beams]).double(), atol=1e-4)
