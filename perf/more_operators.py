"""The two ends of a training step that are timed: the loss over the vocabulary with its gradient, and the update made of the gradients.

  score   losses of given tokens from hidden states and the weight of the head, each by itself        (linear_cross_entropy)
  train   the mean loss, and the gradients of the hidden states and of the weight                      (linear_cross_entropy, its backward pass)
  orth    updates orthogonalised by five Newton-Schulz steps                                            (orthogonalize)

    l = x w^T;  lse_t = log sum_v exp l_tv;  loss_t = lse_t - (1 - e) l_t,target - e / V sum_v l_tv, for tokens whose target is not `IGNORE`
    X = G / (|G| + 1e-7);  A = X X^T;  X <- a X + (b A + c A^2) X, on the side of G's shorter dimension

Hidden sizes are those of the benchmark's matrices (1024, 4096, 5120, 8192, 14336) and ragged ones, vocabularies of generic sizes.
"""
import importlib

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100
STEPS, A1, A3, A5, EPS = 5, 3.4445, -4.7750, 2.0315, 1e-7


def listed():
    return [
        # the probability of one token: the weight's bytes are all there is
        dict(name="score_bf16_1x4096_v32000", kind="score", dtype="bf16", tokens=1, cols=4096, vocab=32000, smooth=0.0),
        # a prompt that is scored, over a large vocabulary of an odd size
        dict(name="score_bf16_300x5120_v131071", kind="score", dtype="bf16", tokens=300, cols=5120, vocab=131071, smooth=0.0),
        # long prompts that are scored
        dict(name="score_bf16_8192x4096_v32000", kind="score", dtype="bf16", tokens=8192, cols=4096, vocab=32000, smooth=0.0),
        # a small model's step: launches are most of it
        dict(name="train_f16_64x1024_v8192", kind="train", dtype="f16", tokens=64, cols=1024, vocab=8192, smooth=0.0),
        # ragged everything: rows off 16 bytes, tiles cut in both directions, smoothed labels
        dict(name="train_bf16_777x1031_v50001", kind="train", dtype="bf16", tokens=777, cols=1031, vocab=50001, smooth=0.1),
        # a training step's loss
        dict(name="train_bf16_4096x4096_v32000", kind="train", dtype="bf16", tokens=4096, cols=4096, vocab=32000, smooth=0.0),
        # ... of a wide model over a large vocabulary
        dict(name="train_bf16_2048x8192_v131072", kind="train", dtype="bf16", tokens=2048, cols=8192, vocab=131072, smooth=0.0),
        # the updates of rank-64 factors of a few layers
        dict(name="orth_f32_24_64x1024", kind="orth", dtype="f32", count=24, rows=64, cols=1024),
        # ragged, FP32
        dict(name="orth_f32_1_777x2051", kind="orth", dtype="f32", count=1, rows=777, cols=2051),
        # attention matrices of a few layers with fewer keys than queries
        dict(name="orth_bf16_4_1024x4096", kind="orth", dtype="bf16", count=4, rows=1024, cols=4096),
        # a square matrix
        dict(name="orth_bf16_1_4096x4096", kind="orth", dtype="bf16", count=1, rows=4096, cols=4096),
        # an MLP matrix, tall, in FP32 as an accumulated gradient is
        dict(name="orth_f32_1_14336x4096", kind="orth", dtype="f32", count=1, rows=14336, cols=4096),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["score", "train", "orth"])
    if kind == "orth":
        rows, cols = _log(rng, 16, 8192), _log(rng, 16, 8192)
        short, cost = min(rows, cols), lambda n: n * min(rows, cols) ** 2 * max(rows, cols)
        count = rng.randint(1, 8)
        while count > 1 and cost(count) > 4096 ** 2 * 8192:
            count -= 1
        if cost(1) > 4096 ** 2 * 8192:
            rows = max(16, rows * 4096 // short)
            cols = max(16, cols * 4096 // short)
        return dict(kind=kind, dtype=rng.choice(["f32", "bf16", "f16"]), count=count, rows=rows, cols=cols)
    tokens, cols, vocab = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 300, 131072)
    most = 2048 * 8192 * 65536
    if tokens * cols * vocab > most:
        tokens = max(1, most // (cols * vocab))
    return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), tokens=tokens, cols=cols, vocab=vocab, smooth=rng.choice([0.0, 0.0, 0.1]))


# ---- the plain form -----------------------------------------------------------------------------------------------

def _plain_loss(state):
    c = state["case"]
    x, w, target = state["x"].detach().float(), state["w"].detach().float(), state["target"]
    logits = x @ w.t()
    top = logits.amax(dim=1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(dim=1, keepdim=True)
    live = target != IGNORE
    at = torch.where(live, target, torch.zeros_like(target))[:, None]
    loss = (top + torch.log(total) - (1 - c["smooth"]) * logits.gather(1, at) - c["smooth"] * logits.mean(dim=1, keepdim=True))[:, 0]
    loss = torch.where(live, loss, torch.zeros_like(loss))
    if c["kind"] == "score":
        return loss
    count = live.sum()
    del logits
    p /= total
    p -= c["smooth"] / c["vocab"]
    p.scatter_add_(1, at, torch.full_like(top, c["smooth"] - 1))
    p *= (live / count)[:, None]
    return {"loss": loss.sum() / count, "dx": (p @ w).to(state["x"].dtype), "dw": (p.t() @ x).to(state["w"].dtype)}


def _plain_orth(g):
    x = g.float()
    x = x.transpose(-2, -1) if x.shape[-2] > x.shape[-1] else x
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        a = x @ x.transpose(-2, -1)
        x = A1 * x + (A3 * a + A5 * (a @ a)) @ x
    return (x.transpose(-2, -1) if g.shape[-2] > g.shape[-1] else x).to(torch.bfloat16)


def _plain(state):
    if state["case"]["kind"] != "orth":
        return _plain_loss(state)
    return list(_plain_orth(torch.stack(state["grads"])).unbind(0))


# ---- what a user's program does ------------------------------------------------------------------------------------

def _ours(state):
    ops = importlib.import_module("bitsqueeze-llm_b200.torch_ops")
    c = state["case"]
    if c["kind"] == "orth":
        return ops.orthogonalize(state["grads"])
    x, w = state["x"], state["w"]
    if c["kind"] == "score":
        return ops.linear_cross_entropy(x, w, state["target"], ignore_index=IGNORE, label_smoothing=c["smooth"], reduction="none")
    loss = ops.linear_cross_entropy(x, w, state["target"], ignore_index=IGNORE, label_smoothing=c["smooth"])
    dx, dw = torch.autograd.grad(loss, (x, w))
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def run(state):
    return _ours(state) if own else _plain(state)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    dtype = DTYPE[case["dtype"]]
    if case["kind"] == "orth":
        rows, cols = case["rows"], case["cols"]
        state["grads"] = []
        for _ in range(case["count"]):
            # a gradient: a few directions that all tokens share, and noise
            g = torch.randn((rows, cols), generator=gen, device="cuda")
            u, v = torch.randn((rows, 4), generator=gen, device="cuda"), torch.randn((4, cols), generator=gen, device="cuda")
            state["grads"].append(((g + u @ v) * 1e-3).to(dtype))
        return state
    tokens, cols, vocab = case["tokens"], case["cols"], case["vocab"]
    w = torch.randn((vocab, cols), generator=gen, device="cuda") * (1.5 / cols ** 0.5)
    target = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    x = torch.randn((tokens, cols), generator=gen, device="cuda")
    # a model that has learned something: the target's logit is 0 to 12 above the others
    lift = 12 * torch.rand((tokens, 1), generator=gen, device="cuda")
    x += w[target] * (lift / 2.25)
    if tokens > 1:                                             # padding and prompts do not count
        target[torch.rand(tokens, generator=gen, device="cuda") < 0.1] = IGNORE
        target[0] = vocab - 1
    state["x"], state["w"], state["target"] = x.to(dtype), w.to(dtype), target
    if case["kind"] == "train":
        state["x"].requires_grad_()
        state["w"].requires_grad_()
    return state


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if case["kind"] == "orth":
        s, l = min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
        return {"bytes": case["count"] * s * l * (size + 2), "flops": case["count"] * STEPS * (s * s * l + s * s * s + 2 * s * s * l)}
    tokens, cols, vocab = case["tokens"], case["cols"], case["vocab"]
    read = (tokens + vocab) * cols * size
    if case["kind"] == "score":
        return {"bytes": read + 12 * tokens, "flops": 2 * tokens * cols * vocab}
    # logits that are not kept are computed again
    return {"bytes": 2 * read + 8 * tokens, "flops": 8 * tokens * cols * vocab}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "orth":
        outs = []
        for g in state["grads"]:
            x = g.double() / (torch.linalg.matrix_norm(g.double()) + EPS)
            for _ in range(STEPS):
                if x.shape[0] <= x.shape[1]:
                    a = x @ x.mT
                    ax = a @ x
                    x = A1 * x + A3 * ax + A5 * (a @ ax)
                else:
                    a = x.mT @ x
                    xa = x @ a
                    x = A1 * x + A3 * xa + A5 * (xa @ a)
            outs.append(x)
        return outs
    e, vocab, target = case["smooth"], case["vocab"], state["target"]
    x, w = state["x"].detach().double(), state["w"].detach().double()
    live = target != IGNORE
    logp = torch.log_softmax(x @ w.mT, dim=1)
    want = torch.full_like(logp, e / vocab)
    want[live.nonzero()[:, 0], target[live]] += 1 - e
    loss = -(want * logp).sum(dim=1) * live
    if case["kind"] == "score":
        return loss
    dl = (torch.exp(logp) - want) * (live.double() / live.sum())[:, None]
    return {"loss": loss.sum() / live.sum(), "dx": dl @ w, "dw": dl.mT @ x}
