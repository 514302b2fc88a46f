"""Prompts, single tokens and beams together, as they are used: a stack on pools of slots against the same stack on one request at a time; and what
surrounds the calls: captured and replayed graphs, other streams, gradients through whole blocks, refusals."""
import types

import pytest
import torch
from torch import nn

from tests.helpers import RefShapedBlock
from tests.test_gpu_packed import cu_of, inputs, plain_scan, close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Norm(nn.Module):
    def __init__(self, d, g):
        super().__init__()
        self.eps, self.use_mup = 1e-5, False
        self.weight = nn.Parameter(1 + 0.1 * torch.randn(d, generator=g))


def stack(layers=2, d=32, seed=0):
    g = torch.Generator().manual_seed(seed)
    torch.manual_seed(seed)
    blocks = []
    for _ in range(layers):
        m = nn.Module()
        m.mixer, m.norm = RefShapedBlock(d), Norm(d, g)
        with torch.no_grad():
            m.mixer.dt_proj.bias.copy_(torch.randn(2 * d, generator=g) - 3)
            m.mixer.A_log.add_(0.2 * torch.randn(2 * d, 16, generator=g))
        blocks.append(m)
    s = types.SimpleNamespace(layers=nn.ModuleList(blocks).to(DEV))
    return s


def one_at_a_time(s, x):
    """A request's rows through the whole stack with the dense drop-ins."""
    from mamba_b200 import mamba
    h = x[None]
    for layer in s.layers:
        normed = torch.nn.functional.rms_norm(h, (h.shape[-1],), layer.norm.weight, layer.norm.eps)
        h = mamba.forward(layer.mixer, normed) + h
    return h[0]


def test_prompts_in_chunks_then_tokens():
    """Prompts of several requests in two chunks, then tokens on the slots: the same as each request on its own, of one length."""
    import mamba_b200
    s = stack()
    pool = mamba_b200.StatePool(s, 9)
    g = torch.Generator().manual_seed(1)
    texts = [torch.randn(n, 32, generator=g).to(DEV) for n in (40, 7, 23, 2)]
    cuts = [17, 0, 22, 1]                                  # rows of the first chunk
    slots = torch.tensor([4, 8, 0, 3], device=DEV)
    with torch.no_grad():
        want = [one_at_a_time(s, t) for t in texts]
        got = [[] for _ in texts]
        first = torch.cat([t[:c] for t, c in zip(texts, cuts)])
        y = pool.prompts(first, cu_of(cuts), slots, max_length=max(cuts))
        for r, part in enumerate(y.split(cuts)):
            got[r].append(part)
        ends = [len(t) - 1 for t in texts]                 # the last row comes as a token
        rest = [e - c for e, c in zip(ends, cuts)]
        second = torch.cat([t[c:e] for t, c, e in zip(texts, cuts, ends)] + [torch.randn(5, 32, generator=g).to(DEV)])
        y = pool.prompts(second, cu_of(rest), slots, resume=torch.tensor([c > 0 for c in cuts], device=DEV))
        for r, part in enumerate(y[:sum(rest)].split(rest)):
            got[r].append(part)
        y = pool.step(torch.stack([t[-1] for t in texts] + [texts[0][0]]), torch.cat([slots, torch.tensor([-1], device=DEV)]))
    for r in range(4):
        close(torch.cat(got[r] + [y[r:r + 1]]), want[r], what=f"request {r}")


def test_training_on_packed_documents():
    """Outputs, and gradients of every parameter, of documents packed into one row: the sum over the documents on their own."""
    from mamba_b200 import mamba
    s, lengths = stack(), [33, 1, 70, 16]
    g = torch.Generator().manual_seed(2)
    x, dy = torch.randn(sum(lengths), 32, generator=g).to(DEV), torch.randn(sum(lengths), 32, generator=g).to(DEV)
    params = list(s.layers.parameters())
    a = x.clone().requires_grad_()
    y = mamba.stack_packed(s, a, cu_of(lengths), max_length=max(lengths))
    got = torch.autograd.grad(y, [a] + params, dy)
    b = x.clone().requires_grad_()
    want_y = torch.cat([one_at_a_time(s, t) for t in b.split(lengths)])
    want = torch.autograd.grad(want_y, [b] + params, dy)
    close(y, want_y, what="y")
    for i, (u, v) in enumerate(zip(got, want)):
        bound = 1e-4 * v.abs().max()                       # two ways through float32 products of two layers
        assert (u - v).abs().max() <= bound, i


def test_gradient_against_differences():
    """The scan's gradients along a random direction, against central differences of the plain scan in 64 bits."""
    import mamba_b200
    lengths, W = [9, 30, 4], 24
    t = inputs(5, sum(lengths), W)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    dy = torch.randn(sum(lengths), W, generator=torch.Generator().manual_seed(6)).to(DEV)
    y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=cu_of(lengths))
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    for i, k in enumerate(leaves):
        d = torch.randn(t[k].shape, generator=torch.Generator().manual_seed(i)).double()
        eps = 1e-5
        values = []
        for sign in (1, -1):
            moved = {n: v.double().cpu() for n, v in t.items()}
            moved[k] = moved[k] + sign * eps * d
            values.append((plain_scan(moved, lengths)[0] * dy.double().cpu()).sum())
        slope = ((values[0] - values[1]) / (2 * eps)).item()
        mine = (grads[k].double().cpu() * d).sum().item()
        scale = (grads[k].double().cpu().abs() * d.abs()).sum().item()
        assert abs(mine - slope) <= 1e-5 * scale, k


def test_captured_and_replayed_with_other_lengths():
    """One graph of a whole step (prompts, tokens, selection, reordering), replayed with other lengths, slots and values."""
    import mamba_b200
    s = stack(1)
    g = torch.Generator().manual_seed(3)
    head = torch.randn(32, 50, generator=g).to(DEV)
    pool, check = mamba_b200.StatePool(s, 8), mamba_b200.StatePool(s, 8)
    x = torch.randn(64, 32, generator=g).to(DEV)
    cu, slots, resume = cu_of([20, 30]), torch.tensor([0, 5], device=DEV), torch.tensor([False, False], device=DEV)
    beams, scores = torch.tensor([[0, 2], [5, 7]], device=DEV), torch.zeros(2, 2, device=DEV)

    def run(p):
        with torch.no_grad():
            y = p.prompts(x, cu, slots, resume)
            z = p.step(x[:4], beams.view(-1))
            best = mamba_b200.beam_select((z @ head).view(2, 2, 50), scores)
            return (y, z, *best, p.reorder(beams, best[2]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(pool)
    torch.cuda.synchronize()
    for t in pool.pools():
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(pool)
    for lengths, where, again in (([20, 30], [0, 5], [False, False]), ([1, 63], [3, 6], [True, False]), ([0, 12], [0, 5], [True, True])):
        x.copy_(torch.randn(64, 32, generator=g))
        cu.copy_(cu_of(lengths))
        slots.copy_(torch.tensor(where))
        resume.copy_(torch.tensor(again))
        graph.replay()
        want = run(check)
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for a, b in zip(pool.pools(), check.pools()):
            assert torch.equal(a, b)


def test_backward_captured_beside_an_eager_one():
    """A captured forward and backward while an eager graph of the same leaves is alive, and two captured ones sharing nothing."""
    import mamba_b200
    lengths = [100, 30, 70]
    t = inputs(1, 200, 64)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    w, b = torch.randn(64, 1, 4, device=DEV, requires_grad=True), torch.randn(64, device=DEV, requires_grad=True)
    cu, dy = cu_of(lengths), torch.randn(200, 64, device=DEV)

    def step():
        x = mamba_b200.causal_conv1d_silu_packed(leaves["x"], w, b, cu_seqlens=cu)
        y = mamba_b200.selective_scan_packed(**{**leaves, "x": x}, cu_seqlens=cu, piece_length=32)
        return y, torch.autograd.grad(y, [*leaves.values(), w, b], dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    x = mamba_b200.causal_conv1d_silu_packed(leaves["x"], w, b, cu_seqlens=cu)
    alive = mamba_b200.selective_scan_packed(**{**leaves, "x": x}, cu_seqlens=cu)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for _, (y, grads) in graphs:
        assert torch.equal(y, want[0])
        for a, c in zip(grads, want[1]):
            close(a, c)                                    # float atomics: order
    torch.autograd.grad(alive.sum(), leaves["x"])


def test_two_streams_at_once():
    """Two calls with workspaces of their own on two streams."""
    import mamba_b200
    lengths = [3000, 200, 100]
    t = [inputs(i, 3300, 96) for i in range(2)]
    cu = cu_of(lengths)
    want = [mamba_b200.selective_scan_packed(**v, cu_seqlens=cu, piece_length=256) for v in t]
    logits, scores = torch.randn(2, 4, 3, 5000, device=DEV), torch.randn(2, 4, 3, device=DEV)
    best = [mamba_b200.beam_select(logits[i], scores[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((mamba_b200.selective_scan_packed(**t[i], cu_seqlens=cu, piece_length=256), mamba_b200.beam_select(logits[i], scores[i])))
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], want[i]) and all(torch.equal(a, b) for a, b in zip(got[i][1], best[i]))


def plain_search(s, embed, head, prompts, K, steps, end):
    """Beam search with every beam's whole text through the dense stack each time."""
    out = []
    for text in prompts:
        beams = [([], 0.0)]
        for _ in range(steps):
            options = []
            for k, (toks, score) in enumerate(beams):
                if end is not None and end in toks:
                    options.append((score, k, end))
                    continue
                x = torch.cat([text, embed[torch.tensor(toks, device=DEV, dtype=torch.long)]]) if toks else text
                with torch.no_grad():
                    logp = torch.log_softmax((one_at_a_time(s, x)[-1] @ head).double(), -1)
                options += [(score + v, k, i) for i, v in enumerate(logp.tolist())]
            options.sort(key=lambda o: (-o[0], o[1], o[2]))
            beams = [(beams[k][0] + [tok], score) for score, k, tok in options[:K]]
        out.append(beams)
    return out


@pytest.mark.parametrize("end", [None, 7])
def test_beam_search(end):
    import mamba_b200
    s, V, G, K, steps = stack(2, 32, 4), 40, 2, 4, 6
    g = torch.Generator().manual_seed(5)
    embed, head = torch.randn(V, 32, generator=g).to(DEV), (0.7 * torch.randn(32, V, generator=g)).to(DEV)
    prompts = [torch.randn(n, 32, generator=g).to(DEV) for n in (11, 5)]
    pool = mamba_b200.StatePool(s, G * K + 1)
    slots = torch.randperm(G * K + 1, generator=g)[: G * K].view(G, K).to(DEV)
    y = pool.prompts(torch.cat(prompts), cu_of([11, 5]), slots[:, 0])
    logits = y[torch.tensor([10, 15], device=DEV)] @ head
    tokens, scores = mamba_b200.beam_search(pool, lambda t: embed[t], lambda h: h @ head, logits, slots, steps, end)
    for r, beams in enumerate(plain_search(s, embed, head, prompts, K, steps, end)):
        assert tokens[r].tolist() == [b[0] for b in beams]
        assert torch.allclose(scores[r].double().cpu(), torch.tensor([b[1] for b in beams]).double(), atol=1e-4)


def test_refusals():
    import mamba_b200
    T, W = 20, 32
    t = inputs(0, T, W)
    cu = cu_of([12, 8])
    scan = lambda **k: mamba_b200.selective_scan_packed(**{**t, "cu_seqlens": cu, **k})
    states, slots = torch.zeros(4, W, 16, device=DEV), torch.tensor([0, 1], device=DEV)
    cases = [(RuntimeError, dict(x=t["x"][None])), (RuntimeError, dict(delta=t["delta"][:5])), (RuntimeError, dict(A=t["A"][:, :8])),
             (RuntimeError, dict(B=t["B"][:, :8])), (RuntimeError, dict(D=t["D"][:5])), (RuntimeError, dict(z=t["z"][:, :8])),
             (RuntimeError, dict(cu_seqlens=cu[None])), (TypeError, dict(cu_seqlens=cu.float())), (RuntimeError, dict(cu_seqlens=cu.cpu())),
             (RuntimeError, dict(states=states)), (RuntimeError, dict(slots=slots)), (RuntimeError, dict(resume=slots > 0)),
             (RuntimeError, dict(states=states, slots=slots[:1])), (TypeError, dict(states=states, slots=slots.float())),
             (TypeError, dict(states=states, slots=slots, resume=slots)), (ValueError, dict(states=states.bfloat16(), slots=slots)),
             (ValueError, dict(states=torch.zeros(8, W, 16, device=DEV)[::2], slots=slots)), (RuntimeError, dict(states=states[:, :8], slots=slots)),
             (RuntimeError, dict(states=states, slots=slots, x=t["x"].clone().requires_grad_())),
             (RuntimeError, dict(states=states.clone().requires_grad_(), slots=slots)),
             (ValueError, dict(piece_length=7)), (ValueError, dict(max_length=-1)), (TypeError, dict(x=t["x"].double()))]
    for error, k in cases:
        with pytest.raises(error):
            scan(**k)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda x: scan(x=x), (t["x"],), (t["x"],))
    conv = lambda **k: mamba_b200.causal_conv1d_silu_packed(**{**dict(x=t["x"], weight=torch.ones(W, 1, 4, device=DEV), cu_seqlens=cu), **k})
    windows = torch.zeros(4, W, 3, device=DEV)
    for error, k in [(RuntimeError, dict(weight=torch.ones(W, 1, 3, device=DEV))), (RuntimeError, dict(weight=torch.ones(5, 1, 4, device=DEV))),
                     (ValueError, dict(windows=windows.bfloat16(), slots=slots)), (RuntimeError, dict(windows=windows[..., :2], slots=slots)),
                     (RuntimeError, dict(x=t["x"].clone().requires_grad_(), windows=windows, slots=slots)), (RuntimeError, dict(windows=windows))]:
        with pytest.raises(error):
            conv(**k)
    rows = dict(x=t["x"][:2], h=states, delta=t["delta"][:2], A=t["A"], B=t["B"][:2], C=t["C"][:2], slots=slots)
    for error, k in [(RuntimeError, dict(slots=slots[:1])), (RuntimeError, dict(h=None)), (ValueError, dict(h=states.bfloat16())),
                     (RuntimeError, dict(delta=t["delta"])), (RuntimeError, dict(B=t["B"])), (TypeError, dict(slots=slots.float()))]:
        with pytest.raises(error):
            mamba_b200.ssm_step_fn(**{**rows, **k})
    logits, scores = torch.zeros(2, 3, 9, device=DEV), torch.zeros(2, 3, device=DEV)
    for error, a, k in [(RuntimeError, (logits[:1], scores), {}), (ValueError, (logits, scores, 0), {}), (ValueError, (logits, scores, 28), {}),
                        (TypeError, (logits, scores.double()), {}), (TypeError, (logits.half(), scores), {}),
                        (ValueError, (logits, scores), dict(finished=scores > 0)), (ValueError, (logits, scores), dict(finished=scores > 0, end_token=9)),
                        (RuntimeError, (logits, scores), dict(finished=scores[:1] > 0, end_token=0)),
                        (RuntimeError, (torch.zeros(1, 65, 9, device=DEV), torch.zeros(1, 65, device=DEV), 1), {}),
                        (RuntimeError, (torch.zeros(1, 3, 99, device=DEV), torch.zeros(1, 3, device=DEV), 65), {}),
                        (RuntimeError, (logits[..., :0], scores), {}), (RuntimeError, (logits.cpu(), scores.cpu()), {})]:
        with pytest.raises(error):
            mamba_b200.beam_select(*a, **k)
    beams = torch.tensor([[0, 1, 2]], device=DEV)
    for error, a in [(RuntimeError, (beams, beams[:, :2], [states])), (TypeError, (beams.float(), beams, [states])), (ValueError, (beams, beams, [states[:, ::2]])),
                     (RuntimeError, (beams, beams, [states, states[:2]])), (RuntimeError, (beams, beams, [states.cpu()])),
                     (RuntimeError, (torch.zeros(1, 65, device=DEV).long(), torch.zeros(1, 65, device=DEV).long(), [states])),
                     (RuntimeError, (beams, beams, [states.clone().requires_grad_()]))]:
        with pytest.raises(error):
            mamba_b200.beam_reorder(*a)


def test_nothing_to_do():
    import mamba_b200
    t = inputs(0, 0, 32)
    y = mamba_b200.selective_scan_packed(**{k: v.clone().requires_grad_() for k, v in t.items()}, cu_seqlens=cu_of([]))
    assert y.shape == (0, 32)
    t = inputs(0, 5, 32)
    assert (mamba_b200.selective_scan_packed(**t, cu_seqlens=cu_of([])) == 0).all()          # rows, but no sequence
    assert (mamba_b200.causal_conv1d_silu_packed(t["x"], torch.ones(32, 1, 4, device=DEV), cu_seqlens=cu_of([0, 0])) == 0).all()
    states, none = torch.ones(2, 32, 16, device=DEV), torch.zeros(0, dtype=torch.long, device=DEV)
    y, _ = mamba_b200.ssm_step_fn(t["x"][:0], states, t["delta"][:0], t["A"], t["B"][:0], t["C"][:0], slots=none)
    assert y.shape == (0, 32) and (states == 1).all()
    s, k, p = mamba_b200.beam_select(torch.zeros(0, 3, 9, device=DEV), torch.zeros(0, 3, device=DEV))
    assert s.shape == k.shape == p.shape == (0, 3)
    assert mamba_b200.beam_reorder(none.view(0, 3), none.view(0, 3), [states]).shape == (0, 3)


def test_wrong_offsets_touch_nothing_else():
    """Offsets that fall, lie outside or repeat: rows and slots around the tensors stay as they are, and nothing faults."""
    import mamba_b200
    T, W = 40, 32
    big = {k: torch.full((T + 20, v.shape[1]), 7.0, device=DEV) for k, v in inputs(0, T, W).items() if v is not None and v.dim() == 2 and v.shape[0] == T}
    t = inputs(0, T, W)
    pool = torch.full((6, W, 16), 3.0, device=DEV)
    for offsets in ([0, 30, 10, 40], [5, 4, 3, 2], [0, 100, 20, 60], [-5, 10, 2000000000, -7], [40, 40, 0, 0]):
        for piece in (0, 16):
            inner = pool[1:5]
            with torch.no_grad():
                y = mamba_b200.selective_scan_packed(**t, cu_seqlens=torch.tensor(offsets, device=DEV), states=inner.clone(),
                                                     slots=torch.tensor([0, -3, 9], device=DEV), piece_length=piece)
                c = mamba_b200.causal_conv1d_silu_packed(t["x"], torch.ones(W, 1, 4, device=DEV), cu_seqlens=torch.tensor(offsets, device=DEV))
            leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
            y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=torch.tensor(offsets, device=DEV), piece_length=piece)
            torch.autograd.grad(y.sum(), list(leaves.values()))
            assert y.shape == c.shape == (T, W)
    torch.cuda.synchronize()
    assert (pool == 3).all() and all((v == 7).all() for v in big.values())
