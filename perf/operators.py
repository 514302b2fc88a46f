"""Operators of serving and of training on packed sequences, as a list of cases that can be timed.

Kinds of case:

  scan      the selective scan over sequences of different lengths laid end to end: prompts whose last states go to the slots of a
            pool (some of them resuming what their slot holds), or documents packed into one row in training, with every gradient
  conv      the causal convolution and SiLU in front of it, likewise
  token     one token of every running request: convolution window, then state update, on the slots of the pools
  select    the best continuations of the beams of several groups, over beams and vocabulary
  reorder   the slots of the beams that go on, and the copies of states where a beam goes on more than once

`own` False computes each in elementary torch operations, `own` True through the package.  d_state is 16 and d_conv 4, as in every
configuration of this repository.
"""
import math
import random

import torch

own = False

N, K = 16, 4
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # Prompts of a batch of requests read by a 2.8b-shaped layer, one of them a single token, one empty, some of them later chunks of a
        # longer prompt; the rows behind the last one are padding of a captured batch.
        {"name": "scan_prompts_2p8b", "kind": "scan", "tokens": 8000, "rows": 8192, "requests": 12, "skew": 1.0, "d_inner": 5120, "dtype": "bf16",
         "train": False},
        # One long prompt among short ones in a 130m-shaped layer: too few channels to fill the GPU unless the long one is cut.
        {"name": "scan_prompts_long", "kind": "scan", "tokens": 16384, "rows": 16384, "requests": 3, "skew": 3.0, "d_inner": 1536, "dtype": "bf16",
         "train": False},
        # Training a 130m-shaped layer on documents packed into one row of tokens.
        {"name": "scan_train_130m", "kind": "scan", "tokens": 16384, "rows": 16384, "requests": 20, "skew": 1.0, "d_inner": 1536, "dtype": "bf16",
         "train": True},
        # Fine-tuning in float32 on a ragged handful of documents and an uneven width.
        {"name": "scan_train_ragged_f32", "kind": "scan", "tokens": 2999, "rows": 2999, "requests": 7, "skew": 1.5, "d_inner": 1000, "dtype": "f32",
         "train": True},
        # The convolution in front of the first scan, and of the training step.
        {"name": "conv_prompts_2p8b", "kind": "conv", "tokens": 8000, "rows": 8192, "requests": 12, "skew": 1.0, "d_inner": 5120, "dtype": "bf16",
         "train": False},
        {"name": "conv_train_ragged_f32", "kind": "conv", "tokens": 2999, "rows": 2999, "requests": 7, "skew": 1.5, "d_inner": 1000, "dtype": "f32",
         "train": True},
        # A decode step of a full batch of a 2.8b-shaped layer, and of three requests of a 130m-shaped one in float32.
        {"name": "token_batch_2p8b", "kind": "token", "requests": 256, "slots": 320, "d_inner": 5120, "dtype": "bf16"},
        {"name": "token_few_f32", "kind": "token", "requests": 3, "slots": 8, "d_inner": 1536, "dtype": "f32"},
        # Beams of a batch of groups over a large vocabulary in bfloat16, and one group over an odd one in float32 whose candidates are
        # twice the beams, so that ended ones can be put aside.
        {"name": "select_batch", "kind": "select", "groups": 64, "beams": 4, "vocab": 50280, "num": 4, "dtype": "bf16"},
        {"name": "select_one_f32", "kind": "select", "groups": 1, "beams": 5, "vocab": 32001, "num": 10, "dtype": "f32"},
        # All 64 layers of a 2.8b shape, eight groups of eight beams of which three go on from another's state; and a small model.
        {"name": "reorder_2p8b", "kind": "reorder", "layers": 64, "groups": 8, "beams": 8, "copied": 3, "slots": 72, "d_inner": 5120,
         "dtype": "bf16"},
        {"name": "reorder_small_f32", "kind": "reorder", "layers": 24, "groups": 1, "beams": 4, "copied": 2, "slots": 6, "d_inner": 1536,
         "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("scan", "scan", "scan", "conv", "token", "select", "reorder"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind in ("scan", "conv"):
        while True:
            width = rng.choice((8 * _log(rng, 4, 640), 32 * _log(rng, 1, 160)))
            requests, tokens = _log(rng, 1, 64), _log(rng, 33, 16384)
            train = rng.random() < 0.4
            if tokens * width <= 16384 * 1536 // (1 if dtype == "bf16" else 2) * (1 if train or kind == "conv" else 2) and requests < tokens:
                break
        rows = tokens + (rng.randrange(1, 200) if rng.random() < 0.5 else 0)
        return {"kind": kind, "tokens": tokens, "rows": rows, "requests": requests, "skew": round(rng.uniform(0.0, 3.0), 2), "d_inner": width,
                "dtype": dtype, "train": train}
    if kind == "token":
        requests = _log(rng, 1, 256)
        return {"kind": kind, "requests": requests, "slots": requests + rng.randrange(0, 40), "d_inner": 8 * _log(rng, 8, 640), "dtype": dtype}
    if kind == "select":
        while True:
            beams, groups, vocab = rng.randrange(1, 17), _log(rng, 1, 128), _log(rng, 33, 128256)
            if beams * groups * vocab <= 64 * 4 * 50280 // (1 if dtype == "bf16" else 2):
                break
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": vocab, "num": min(beams * rng.choice((1, 2)), beams * vocab), "dtype": dtype}
    beams = rng.randrange(2, 13)
    groups, layers, width = _log(rng, 1, 8), _log(rng, 1, 64), 8 * _log(rng, 16, 640)
    slots = groups * beams + rng.randrange(0, 9)
    if slots * layers * width > 72 * 64 * 5120:
        layers = max(1, 72 * 64 * 5120 // (slots * width))
    return {"kind": kind, "layers": layers, "groups": groups, "beams": beams, "copied": rng.randrange(0, beams), "slots": slots, "d_inner": width,
            "dtype": dtype}


# ------------------------------------------------------------------------------------ inputs

def _lengths(case, rng):
    """Lengths of the requests, in the order they come: a large `skew` makes one of them most of the tokens; of eight or more, one has a
    single token and one none."""
    n, tokens = case["requests"], case["tokens"]
    rest = n - 2 if n >= 8 else n
    weights = [math.exp(case["skew"] * random.Random(1000 * n + i).gauss(0, 1)) for i in range(rest)]
    left = tokens - (1 if n >= 8 else 0)
    lengths = [max(1, int(left * w / sum(weights))) for w in weights]
    at = max(range(rest), key=lambda i: lengths[i])
    lengths[at] += left - sum(lengths)
    if n >= 8:
        lengths += [1, 0]
    rng.shuffle(lengths)
    return lengths


def _dt_bias(width, gen):
    """Inverse softplus of dt ~ log-uniform [1e-3, 1e-1], the reference's initialisation."""
    dt = torch.exp(torch.rand(width, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    return dt + torch.log(-torch.expm1(-dt))


def _rates(width, gen):
    """A of a trained model: moved away from -1 .. -N."""
    start = torch.log(torch.arange(1, N + 1, dtype=torch.float32, device="cuda")).repeat(width, 1)
    return -torch.exp(start + 0.2 * torch.randn(width, N, generator=gen, device="cuda"))


def _packed(case, gen, seed):
    """Where the sequences lie, and the slots they go to."""
    rng = random.Random(seed)
    lengths = _lengths(case, rng)
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    slots = rng.sample(range(len(lengths) + 4), len(lengths))
    on = lambda v, t: torch.tensor(v, dtype=t, device="cuda")
    return {"cu_seqlens": on(starts, torch.int32), "max_length": max(lengths), "slots": on(slots, torch.int64),
            "resume": on([rng.random() < 0.5 for _ in lengths], torch.bool), "n_slots": len(lengths) + 4}


def _prepare_scan(case, gen, seed):
    T, W, dtype = case["rows"], case["d_inner"], DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    s = {"x": torch.nn.functional.silu(normal(T, W)).to(dtype), "delta": (normal(T, W) * 0.5).to(dtype), "A": _rates(W, gen),
         "B": normal(T, N).to(dtype), "C": normal(T, N).to(dtype), "D": 1.0 + 0.1 * normal(W), "z": normal(T, W).to(dtype),
         "delta_bias": _dt_bias(W, gen)}
    if case["train"]:
        s = {k: t.requires_grad_() for k, t in s.items()}
        s["dy"] = normal(T, W).to(dtype)
    s.update(_packed(case, gen, seed))
    if not case["train"]:
        s["states"] = normal(s["n_slots"], W, N)
    return s


def _prepare_conv(case, gen, seed):
    T, W, dtype = case["rows"], case["d_inner"], DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    s = {"x": normal(T, W).to(dtype), "weight": 0.5 * normal(W, 1, K), "bias": 0.5 * normal(W)}
    if case["train"]:
        s = {k: t.requires_grad_() for k, t in s.items()}
        s["dy"] = normal(T, W).to(dtype)
    s.update(_packed(case, gen, seed))
    if not case["train"]:
        s["windows"] = normal(s["n_slots"], W, K - 1).to(dtype)
    return s


def _prepare_token(case, gen, seed):
    B, W, dtype = case["requests"], case["d_inner"], DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    slots = random.Random(seed).sample(range(case["slots"]), B)
    # `xc` stands for the convolution's output, so that a value next to a rounding border there is not one in the states here
    return {"x": normal(B, W).to(dtype), "xc": torch.nn.functional.silu(normal(B, W)).to(dtype), "delta": (normal(B, W) * 0.5).to(dtype),
            "A": _rates(W, gen), "B": normal(B, N).to(dtype), "C": normal(B, N).to(dtype), "D": 1.0 + 0.1 * normal(W), "z": normal(B, W).to(dtype), "delta_bias": _dt_bias(W, gen),
            "weight": 0.5 * normal(W, 1, K), "bias": 0.5 * normal(W), "states": normal(case["slots"], W, N),
            "windows": normal(case["slots"], W, K - 1).to(dtype), "slots": torch.tensor(slots, dtype=torch.int64, device="cuda")}


def _prepare_select(case, gen, seed):
    G, B, V, dtype = case["groups"], case["beams"], case["vocab"], DTYPES[case["dtype"]]
    logits = (3.0 * torch.randn(G, B, V, generator=gen, device="cuda")).to(dtype)
    scores = -20.0 * torch.rand(G, B, generator=gen, device="cuda")
    finished = torch.rand(G, B, generator=gen, device="cuda") < 0.15
    return {"logits": logits, "scores": scores, "finished": finished, "end": 2, "num": case["num"]}


def _prepare_reorder(case, gen, seed):
    G, B, W, dtype = case["groups"], case["beams"], case["d_inner"], DTYPES[case["dtype"]]
    rng = random.Random(seed)
    slots = rng.sample(range(case["slots"]), G * B)
    parents = []
    for _ in range(G):                                    # all but `copied` beams go on, some of them more than once
        on = rng.sample(range(B), B - case["copied"])
        group = on + [rng.choice(on) for _ in range(case["copied"])]
        rng.shuffle(group)
        parents.append(group)
    return {"slots": torch.tensor(slots, dtype=torch.int64, device="cuda").view(G, B),
            "parents": torch.tensor(parents, dtype=torch.int64, device="cuda"),
            "states": torch.randn(case["layers"], case["slots"], W, N, generator=gen, device="cuda"),
            "windows": torch.randn(case["layers"], case["slots"], W, K - 1, generator=gen, device="cuda").to(dtype)}


_PREPARE = {"scan": _prepare_scan, "conv": _prepare_conv, "token": _prepare_token, "select": _prepare_select, "reorder": _prepare_reorder}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"kind": case["kind"], **_PREPARE[case["kind"]](case, gen, seed)}


# ------------------------------------------------------------------------------------ plain forms

def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _silu(v):
    return v / (1 + torch.exp(-v))


def _places(s, rows):
    """Of every row: its sequence, its place in it, and whether it belongs to one."""
    cu = s["cu_seqlens"].long()
    t = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    inside = t < cu[-1]
    seq = torch.clamp(seq, max=cu.numel() - 2)
    return cu, seq, t - cu[seq], inside


def _linear_scan(a, u, longest):
    """h[t] = a[t] h[t-1] + u[t] along the first dimension, in steps that double."""
    d = 1
    while d < longest:
        u = torch.cat([u[:d], torch.addcmul(u[d:], a[d:], u[:-d])])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return u


def _plain_scan_values(s, h0):
    x, delta, B, C, z = (s[k].detach().float() for k in ("x", "delta", "B", "C", "z"))
    A, D, bias = s["A"].detach(), s["D"].detach(), s["delta_bias"].detach()
    cu, seq, place, inside = _places(s, x.shape[0])
    raw = delta + bias
    dt = _softplus(raw) * inside[:, None]
    x = torch.where(inside[:, None], x, 0.0)
    a = torch.exp(dt[..., None] * A)
    u = (dt * x)[..., None] * B[:, None, :]
    # nothing is carried into a first token but the state that its sequence resumes
    first = (place == 0) & inside
    carried = a
    a = torch.where(first[:, None, None], 0.0, a)
    if h0 is not None:
        begins = torch.nonzero_static(first, size=cu.numel() - 1, fill_value=0)[:, 0]
        full = (cu[1:] > cu[:-1])
        # sequences without tokens begin nowhere: theirs are left out by a weight of zero
        rank = torch.cumsum(full.long(), 0) - 1
        at = begins[torch.clamp(rank, min=0)]
        u.index_add_(0, at, carried[at] * h0 * full[:, None, None])
    h = _linear_scan(a, u, s["max_length"])
    y = (h * C[:, None, :]).sum(-1) + D * x
    return x, dt, raw, B, C, z, A, D, a, h, y, cu, inside


def _plain_scan(s):
    kind = s["x"].dtype
    if "dy" not in s:
        old = s["states"][s["slots"]]
        h0 = old * s["resume"][:, None, None]
        _, _, _, _, _, z, _, _, _, h, y, cu, inside = _plain_scan_values(s, h0)
        full = cu[1:] > cu[:-1]
        last = h[torch.clamp(cu[1:] - 1, min=0)]
        s["states"].index_copy_(0, s["slots"], torch.where(full[:, None, None], last, old))
        return (y * _silu(z) * inside[:, None]).to(kind), s["states"]
    x, dt, raw, B, C, z, A, D, a, h, y, cu, inside = _plain_scan_values(s, None)
    gate = _silu(z)
    dy = s["dy"].float() * inside[:, None]
    sig = 1 / (1 + torch.exp(-z))
    dz = dy * y * sig * (1 + z * (1 - sig))
    dyg = dy * gate
    # g[t] = dy'[t] C[t] + a[t+1] g[t+1]: the same scan from the end, with the decays one place on
    after = torch.cat([a[1:], torch.zeros_like(a[:1])])
    g = _linear_scan(after.flip(0), (dyg[..., None] * C[:, None, :]).flip(0), s["max_length"]).flip(0)
    del after
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    w = g * a * before                                    # a is 0 at first tokens, where nothing came before
    gB = (g * B[:, None, :]).sum(-1)
    dA = (w * dt[..., None]).sum(0)
    ddt = (w * A).sum(-1) + x * gB
    dx = dt * gB + dyg * D
    dB = torch.einsum("ten,te->tn", g, dt * x)
    dC = torch.einsum("ten,te->tn", h, dyg)
    draw = ddt / (1 + torch.exp(-raw)) * inside[:, None]
    out = (y * gate * inside[:, None]).to(kind)
    to = lambda v: (v * inside[:, None]).to(kind)
    return out, (to(dx), draw.to(kind), dA, to(dB), to(dC), (dyg * x).sum(0), to(dz), draw.sum(0))


def _plain_conv(s):
    kind, x, w = s["x"].dtype, s["x"].detach().float(), s["weight"].detach()[:, 0]
    cu, seq, place, inside = _places(s, x.shape[0])
    x = torch.where(inside[:, None], x, 0.0)
    serving = "dy" not in s
    if serving:
        old = s["windows"][s["slots"]].float()
        window = old * s["resume"][:, None, None]
    taps = []
    for k in range(K):
        back = K - 1 - k                                  # this tap looks so far back
        moved = torch.cat([torch.zeros_like(x[:back]), x[: x.shape[0] - back]])
        before = place < back
        if serving:
            head = window[seq, :, torch.clamp(place + k, max=K - 2)]
            taps.append(torch.where(before[:, None], head, moved))
        else:
            taps.append(torch.where(before[:, None], 0.0, moved))
    pre = s["bias"].detach() + sum(w[:, k] * taps[k] for k in range(K))
    y = (_silu(pre) * inside[:, None]).to(kind)
    if serving:
        lengths = cu[1:] - cu[:-1]
        j = torch.arange(K - 1, device="cuda")
        place_of = lengths[:, None] - (K - 1) + j         # place of the input that goes to entry j; before the first token: the old window
        rows = torch.clamp(cu[:-1, None] + place_of, min=0)
        fresh = x[rows].transpose(1, 2)
        kept = torch.gather(window, 2, torch.clamp(lengths[:, None] + j, max=K - 2)[:, None, :].expand(-1, x.shape[1], -1))
        new = torch.where((place_of >= 0)[:, None, :], fresh, kept)
        new = torch.where((lengths > 0)[:, None, None], new, old)
        s["windows"].index_copy_(0, s["slots"], new.to(kind))
        return y, s["windows"]
    sig = 1 / (1 + torch.exp(-pre))
    dpre = s["dy"].float() * inside[:, None] * sig * (1 + pre * (1 - sig))
    left = cu[seq + 1] - torch.arange(x.shape[0], device="cuda")          # tokens of the sequence from this one on
    dx = sum(w[:, k] * torch.where((left > K - 1 - k)[:, None], torch.cat([dpre[K - 1 - k:], torch.zeros_like(dpre[:K - 1 - k])]), 0.0)
             for k in range(K))
    dw = torch.stack([(dpre * taps[k]).sum(0) for k in range(K)], 1)[:, None]
    return y, ((dx * inside[:, None]).to(kind), dw, dpre.sum(0))


def _plain_token(s):
    kind, slots = s["x"].dtype, s["slots"]
    window = torch.cat([s["windows"][slots], s["x"][..., None]], 2)
    pre = (window.float() * s["weight"][:, 0]).sum(-1) + s["bias"]
    convolved = _silu(pre).to(kind)
    s["windows"].index_copy_(0, slots, window[..., 1:])
    x, delta, B, C, z = (s[k].float() for k in ("xc", "delta", "B", "C", "z"))
    dt = _softplus(delta + s["delta_bias"])
    h = torch.exp(dt[..., None] * s["A"]) * s["states"][slots] + (dt * x)[..., None] * B[:, None, :]
    s["states"].index_copy_(0, slots, h)
    y = ((h * C[:, None, :]).sum(-1) + s["D"] * x) * _silu(z)
    return convolved, y.to(kind), s["windows"], s["states"]


def _plain_select(s):
    # in 64 bits: candidates of different beams that are next to each other have to come out in their order
    logits, G, B, V = s["logits"].double(), *s["logits"].shape
    top = logits.max(-1, keepdim=True).values
    total = top + torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    value = s["scores"].double()[..., None] + (logits - total)
    ends = torch.arange(V, device="cuda") == s["end"]
    value = torch.where(s["finished"][..., None], torch.where(ends, s["scores"].double()[..., None], -math.inf), value)
    value = torch.where(torch.isnan(value), -math.inf, value).view(G, B * V)
    order = torch.sort(value, dim=-1, descending=True, stable=True)
    best, at = order.values[:, : s["num"]], order.indices[:, : s["num"]]
    return best.float(), at % V, at // V


def _plain_reorder(s):
    slots, parents = s["slots"], s["parents"]
    B = slots.shape[1]
    same = parents[:, :, None] == parents[:, None, :]
    first = ~torch.tril(same, -1).any(-1)                 # the lowest child of its parent
    going_on = (parents[:, None, :] == torch.arange(B, device="cuda")[:, None]).any(-1)
    free = torch.argsort(going_on.long(), dim=1, stable=True)             # beams without children first
    rank = torch.cumsum((~first).long(), 1) - 1
    new = torch.where(first, slots.gather(1, parents), slots.gather(1, free.gather(1, torch.clamp(rank, min=0))))
    source = slots.gather(1, parents).view(-1)
    for pool in (s["states"], s["windows"]):
        pool.index_copy_(1, new.view(-1), pool.index_select(1, source))
    return new, s["states"], s["windows"]


# ------------------------------------------------------------------------------------ the package's calls

def _own_scan(s):
    import mamba_b200
    args = (s["x"], s["delta"], s["A"], s["B"], s["C"], s["D"])
    if "dy" not in s:
        with torch.no_grad():
            y = mamba_b200.selective_scan_packed(*args, z=s["z"], delta_bias=s["delta_bias"], cu_seqlens=s["cu_seqlens"], states=s["states"],
                                                 slots=s["slots"], resume=s["resume"], max_length=s["max_length"])
        return y, s["states"]
    y = mamba_b200.selective_scan_packed(*args, z=s["z"], delta_bias=s["delta_bias"], cu_seqlens=s["cu_seqlens"], max_length=s["max_length"])
    wanted = (*args, s["z"], s["delta_bias"])
    return y.detach(), torch.autograd.grad(y, wanted, s["dy"])


def _own_conv(s):
    import mamba_b200
    if "dy" not in s:
        with torch.no_grad():
            y = mamba_b200.causal_conv1d_silu_packed(s["x"], s["weight"], s["bias"], cu_seqlens=s["cu_seqlens"], windows=s["windows"],
                                                     slots=s["slots"], resume=s["resume"])
        return y, s["windows"]
    y = mamba_b200.causal_conv1d_silu_packed(s["x"], s["weight"], s["bias"], cu_seqlens=s["cu_seqlens"])
    return y.detach(), torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])


def _own_token(s):
    import mamba_b200
    with torch.no_grad():
        convolved, _ = mamba_b200.conv_step_fn(s["x"], s["windows"], s["weight"], s["bias"], slots=s["slots"])
        y, _ = mamba_b200.ssm_step_fn(s["xc"], s["states"], s["delta"], s["A"], s["B"], s["C"], s["D"], z=s["z"], delta_bias=s["delta_bias"],
                                      slots=s["slots"])
    return convolved, y, s["windows"], s["states"]


def _own_select(s):
    import mamba_b200
    return mamba_b200.beam_select(s["logits"], s["scores"], s["num"], finished=s["finished"], end_token=s["end"])


def _own_reorder(s):
    import mamba_b200
    pools = [*s["states"].unbind(0), *s["windows"].unbind(0)]
    return mamba_b200.beam_reorder(s["slots"], s["parents"], pools), s["states"], s["windows"]


_PLAIN = {"scan": _plain_scan, "conv": _plain_conv, "token": _plain_token, "select": _plain_select, "reorder": _plain_reorder}
_OWN = {"scan": _own_scan, "conv": _own_conv, "token": _own_token, "select": _own_select, "reorder": _own_reorder}


def run(state):
    if own:
        return _OWN[state["kind"]](state)
    with torch.no_grad():
        return _PLAIN[state["kind"]](state)


# ------------------------------------------------------------------------------------ work

def work(case):
    """Each input read once, each output written once.  Operations: 8 per state element of a scan forward (exponential, its argument,
    input, recurrence, contraction), 22 backward; 2 per tap of the convolution; 2 per logit."""
    e = 2 if case["dtype"] == "bf16" else 4
    kind = case["kind"]
    if kind in ("scan", "conv"):
        T, R, W = case["tokens"], case["requests"], case["d_inner"]
    if kind == "scan":
        params = 4 * W * (N + 2)
        if case["train"]:
            return {"bytes": T * (8 * W + 4 * N) * e + 2 * params, "flops": 30 * T * W * N}
        return {"bytes": T * (4 * W + 2 * N) * e + params + 6 * R * W * N, "flops": 8 * T * W * N}
    if kind == "conv":
        params = 4 * W * (K + 1)
        if case["train"]:
            return {"bytes": 4 * T * W * e + 2 * params, "flops": 8 * K * T * W}
        return {"bytes": 2 * T * W * e + params + 3 * R * W * (K - 1) * e // 2, "flops": 2 * K * T * W}
    if kind == "token":
        B, W = case["requests"], case["d_inner"]
        return {"bytes": 2 * B * W * (4 * N + (K - 1) * e) + 6 * B * W * e + 4 * W * (N + K + 3), "flops": B * W * (8 * N + 2 * K)}
    if kind == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": n * e, "flops": 2 * n}
    state = case["d_inner"] * (4 * N + (K - 1) * e)
    n = case["groups"] * case["copied"]
    return {"bytes": 2 * case["layers"] * n * state + 24 * case["groups"] * case["beams"], "flops": 0}


# ------------------------------------------------------------------------------------ 64 bits, one token after the other

def _in_turn(lengths, starts):
    """Rows in the order first tokens, second tokens, ...; how many there are of each; and the sequences, longest first."""
    order = sorted(range(len(lengths)), key=lambda r: -lengths[r])
    rows, counts = [], []
    for t in range(max(lengths)):
        live = [r for r in order if lengths[r] > t]
        rows += [starts[r] + t for r in live]
        counts.append(len(live))
    return rows, counts, order


def _exact_scan(s):
    f = torch.nn.functional
    starts = s["cu_seqlens"].tolist()
    lengths = [b - a for a, b in zip(starts, starts[1:])]
    rows, counts, order = _in_turn(lengths, starts)
    rows = torch.tensor(rows, device="cuda")
    T = s["x"].shape[0]
    names = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias")
    train = "dy" in s
    v = {k: s[k].detach().double().requires_grad_(train) for k in names}
    x, dt, B, C, z = v["x"][rows], f.softplus(v["delta"][rows] + v["delta_bias"], threshold=1e9), v["B"][rows], v["C"][rows], v["z"][rows]
    decay = torch.exp(dt.unsqueeze(-1) * v["A"]).split(counts)
    new = (dt * x).unsqueeze(-1).mul(B.unsqueeze(1)).split(counts)
    if train:
        h = torch.zeros(counts[0], x.shape[1], N, dtype=torch.float64, device="cuda")
    else:
        at = torch.tensor(order, device="cuda")[: counts[0]]
        h = s["states"].double()[s["slots"][at]] * s["resume"][at].double()[:, None, None]
    hs = []
    for t, n in enumerate(counts):
        h = decay[t] * h[:n] + new[t]
        hs.append(h)
    y = (torch.einsum("ten,tn->te", torch.cat(hs), C) + v["D"] * x) * f.silu(z)
    y = torch.zeros(T, x.shape[1], dtype=torch.float64, device="cuda").index_copy(0, rows, y)
    if train:
        return y.detach(), torch.autograd.grad(y, [v[k] for k in names], s["dy"].double())
    states = s["states"].double()
    for t, n in enumerate(counts):
        ended = counts[t + 1] if t + 1 < len(counts) else 0
        for i in range(ended, n):
            states[s["slots"][order[i]]] = hs[t][i]
    return y, states


def _exact_conv(s):
    f = torch.nn.functional
    starts = s["cu_seqlens"].tolist()
    train = "dy" in s
    x, w, b = (s[k].detach().double().requires_grad_(train) for k in ("x", "weight", "bias"))
    ys, windows = [], None if train else s["windows"].double()
    for r, (lo, hi) in enumerate(zip(starts, starts[1:])):
        if lo == hi:
            continue
        head = torch.zeros(K - 1, x.shape[1], dtype=torch.float64, device="cuda")
        if not train and bool(s["resume"][r]):
            head = windows[s["slots"][r]].t().clone()
        line = torch.cat([head, x[lo:hi]])
        ys.append(f.silu(f.conv1d(line.t()[None], w, b, groups=x.shape[1])[0].t()))
        if not train:
            windows[s["slots"][r]] = line[-(K - 1):].t()
    y = torch.cat(ys + [torch.zeros(x.shape[0] - starts[-1], x.shape[1], dtype=torch.float64, device="cuda")])
    if train:
        return y.detach(), torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return y, windows


def _exact_token(s):
    f = torch.nn.functional
    d = {k: t.double() if t.is_floating_point() else t for k, t in s.items() if k != "kind"}
    convolved, y, windows, states = [], [], d["windows"].clone(), d["states"].clone()
    for i, slot in enumerate(d["slots"].tolist()):
        line = torch.cat([windows[slot], d["x"][i][:, None]], 1)
        convolved.append(f.silu(torch.einsum("ek,ek->e", line, d["weight"][:, 0]) + d["bias"]))
        windows[slot] = line[:, 1:]
        c = d["xc"][i]
        dt = f.softplus(d["delta"][i] + d["delta_bias"], threshold=1e9)
        states[slot] = states[slot] * torch.exp(torch.outer(dt, torch.ones(N, device="cuda").double()) * d["A"]) + torch.outer(dt * c, d["B"][i])
        y.append((states[slot] @ d["C"][i] + d["D"] * c) * f.silu(d["z"][i]))
    return torch.stack(convolved), torch.stack(y), windows, states


def _exact_select(s):
    best = []
    for g in range(s["logits"].shape[0]):
        value = torch.log_softmax(s["logits"][g].double(), -1) + s["scores"][g].double()[:, None]
        for k in torch.nonzero(s["finished"][g])[:, 0].tolist():
            value[k] = -math.inf
            value[k, s["end"]] = s["scores"][g, k].double()
        best.append(torch.topk(value.view(-1), s["num"]).values)
    return torch.stack(best), None, None


def _exact_reorder(s):
    states, windows = s["states"].clone(), s["windows"].clone()
    for slots, parents in zip(s["slots"].tolist(), s["parents"].tolist()):
        spare = [slots[k] for k in range(len(slots)) if k not in parents]
        seen = set()
        for p in parents:
            if p in seen:
                to = spare.pop(0)
                states[:, to], windows[:, to] = s["states"][:, slots[p]], s["windows"][:, slots[p]]
            seen.add(p)
    return None, states, windows


_EXACT = {"scan": _exact_scan, "conv": _exact_conv, "token": _exact_token, "select": _exact_select, "reorder": _exact_reorder}


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))
