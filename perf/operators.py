"""What is timed of the operators that adapt and train a layer: low-rank adapters of many requests beside a shared projection,
with their gradients, and the balance loss of a router with per-expert counts and the gradient of the router's logits.

Shapes: the projections of the layer that the benchmark's configurations name (hidden 2048, shared intermediate 512, 512
experts, top 10), of the Qwen3.8 checkpoint's layer (hidden 2560, intermediate 640), and a square one of the hidden size.
Activations are FP32, as everywhere in this framework; adapters F32, F16 or BF16.

Adapters: y = base + scale_a B_a (A_a x) for every token's adapter a; tokens without one keep base.  A prompt's tokens lie
together (one request after another), decode steps have one token a request.  Balance: with p = softmax(logits), c the
number of (token, slot) pairs of each expert, P the sum of p over the N tokens that the mask leaves,
loss = experts / N^2 sum_e c_e P_e.
"""
from __future__ import annotations

import math

import torch

own = False

GGUF = {"F32": 0, "F16": 1, "BF16": 30}
DTYPE = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
NONE = -1                                       # slot of a token without an adapter (0xffffffff)


def adapter_case(name, op, tokens, k, n, rank, slots, dtype, requests):
    c = {"op": op, "tokens": tokens, "k": k, "n": n, "rank": rank, "slots": slots, "dtype": dtype, "requests": requests}
    return dict(c, name=name) if name else c


def balance_case(name, op, tokens, experts, top_k, spread, padded, norm):
    c = {"op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "spread": spread, "padded": padded, "norm": norm}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one stream, one token: the shared expert's gate beside its adapter, latency alone
        adapter_case("adapters decode-1", "adapter forward", 1, 2048, 512, 16, 4, "BF16", 1),
        # 64 streams at one token each, of 48 adapters
        adapter_case("adapters serve-64", "adapter forward", 64, 2048, 2048, 32, 48, "BF16", 64),
        # prompts of five requests in one chunk on the checkpoint's layer, odd length and rank
        adapter_case("adapters prefill-777", "adapter forward", 777, 2560, 640, 20, 7, "F16", 5),
        # long prompts of eight requests
        adapter_case("adapters prefill-8192", "adapter forward", 8192, 2048, 2048, 64, 8, "BF16", 8),
        # a small fine-tuning step on the down projection
        adapter_case("adapters train-333", "adapter backward", 333, 512, 2048, 8, 2, "F32", 3),
        # a step on the router or a gate projection, FP32 master weights
        adapter_case("adapters train-4096", "adapter backward", 4096, 2048, 512, 16, 4, "F32", 16),
        # the largest step
        adapter_case("adapters train-8192", "adapter backward", 8192, 2048, 2048, 64, 3, "BF16", 11),
        # load of a decode step of 64 streams
        balance_case("balance serve-64", "balance forward", 64, 512, 10, 1.0, 0.0, True),
        # the routers of 48 layers over a chunk of 1024 tokens in one loss
        balance_case("balance stack-49152", "balance forward", 49152, 512, 10, 1.0, 0.0, True),
        # gradients: a padded micro-batch of a small router, a batch of eight sequences, and the stack
        balance_case("balance grad-1000", "balance backward", 1000, 60, 4, 2.0, 0.3, False),
        balance_case("balance grad-8192", "balance backward", 8192, 512, 10, 1.0, 0.1, True),
        balance_case("balance grad-49152", "balance backward", 49152, 512, 10, 1.0, 0.0, True),
    ]


def log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    """Any batch from one token up, any projection of the two layers, odd ranks and expert counts."""
    op = rng.choice(["adapter forward", "adapter backward", "balance forward", "balance backward"])
    if op.startswith("adapter"):
        k, n = rng.choice([(2048, 512), (512, 2048), (2048, 2048), (2560, 640), (640, 2560), (1000, 333), (777, 1030)])
        tokens, slots = log_int(rng, 1, 8192), log_int(rng, 1, 48)
        rank = min(64, max(1, rng.choice([4, 8, 16, 32, 64, log_int(rng, 1, 64)])))
        if tokens * slots * rank > 8192 * 8 * 64:                                   # plain forms compute every slot for every token
            slots = max(1, 8192 * 8 * 64 // (tokens * rank))
        requests = tokens if tokens <= 64 and rng.random() < 0.5 else log_int(rng, 1, min(tokens, 32))
        return adapter_case(None, op, tokens, k, n, rank, slots, rng.choice(["F32", "F16", "BF16"]), requests)
    experts = rng.choice([512, 512, 128, 60, 7, log_int(rng, 8, 1024)])
    tokens = log_int(rng, 1, 49152 * 512 // max(512, experts))
    return balance_case(None, op, tokens, experts, min(experts, rng.choice([1, 2, 4, 8, 10])), rng.choice([0.3, 1.0, 3.0]),
                        rng.choice([0.0, 0.0, 0.2, 0.7]), rng.random() < 0.7)


class State:
    """The inputs and output buffers of one case, and where the framework's operators are called the workspace."""


def slot_ids(case, gen):
    """The adapter of every token: `requests` runs of tokens one after another, each request with an adapter or (one in eight) none."""
    t, q = case["tokens"], case["requests"]
    cuts = torch.randperm(max(t - 1, 1), generator=gen, device="cuda")[:q - 1] + 1 if q > 1 else torch.empty(0, device="cuda", dtype=torch.long)
    request = torch.zeros(t, device="cuda", dtype=torch.long)
    request[cuts] = 1
    request = request.cumsum(0)
    of = torch.randint(0, case["slots"], (q,), generator=gen, device="cuda")
    of[torch.rand(q, generator=gen, device="cuda") < 0.125] = NONE
    of[0] = of[0].clamp(min=0)                                                      # never a batch without any
    return of[request].to(torch.int32)


def workspace(case):
    from picoforge_b200 import abi, tuning
    api = abi.product()
    api.lib.qw4cu_set_stream(torch.cuda.current_stream().cuda_stream or 1)          # 1: the legacy default stream by its handle
    if case["op"].startswith("adapter"):
        return tuning.TuneWork(api, tokens=case["tokens"], slots=case["slots"], rank=case["rank"])
    return tuning.TuneWork(api, tokens=case["tokens"], experts=case["experts"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = State()
    s.case, t = case, case["tokens"]
    if case["op"].startswith("adapter"):
        k, n, r, slots, dtype = case["k"], case["n"], case["rank"], case["slots"], DTYPE[case["dtype"]]
        s.x, s.slot = normal(t, k), slot_ids(case, gen)
        s.a, s.b = (normal(slots, r, k) * k ** -0.5).to(dtype), (normal(slots, n, r) * 0.1).to(dtype)
        s.scale = 0.5 + 1.5 * torch.rand(slots, generator=gen, device="cuda")
        if case["op"] == "adapter forward":
            s.base = normal(t, n)                                                   # what the shared projection gave
            s.out = {"y": torch.empty(t, n, device="cuda")}
        else:
            s.dy, s.base = normal(t, n) * 0.05, normal(t, k) * 0.05                 # base: the gradient through the shared projection
            s.out = {"dx": torch.empty(t, k, device="cuda"), "da": torch.empty(slots, r, k, device="cuda"), "db": torch.empty(slots, n, r, device="cuda")}
    else:
        e, top = case["experts"], case["top_k"]
        popularity = -0.6 * torch.log(torch.randperm(e, generator=gen, device="cuda").float() + 1.0)
        s.logits = case["spread"] * normal(t, e) + popularity
        s.ids = s.logits.topk(top, dim=1).indices.to(torch.int32)
        s.mask = None
        if case["padded"]:
            s.mask = (torch.rand(t, generator=gen, device="cuda") >= case["padded"]).to(torch.uint8)
            s.mask[0] = 1
            s.logits[s.mask == 0] = float("nan")                                    # rows of padding hold anything
            s.ids[s.mask == 0] = 0
        if case["op"] == "balance forward":
            s.out = {"counts": torch.empty(e + 1, device="cuda", dtype=torch.int32), "prob_sums": torch.empty(e, device="cuda"),
                     "loss": torch.empty(1, device="cuda")}
        else:
            valid = torch.ones(t, device="cuda", dtype=torch.bool) if s.mask is None else s.mask.bool()
            s.counts = torch.cat([torch.bincount(s.ids[valid].long().reshape(-1), minlength=e), valid.sum()[None]]).to(torch.int32)
            s.weights_grad, s.loss_grad = normal(t, top) * (0.02 / t), 0.01
            s.out = {"grad": torch.empty(t, e, device="cuda")}
    if own:
        s.work = workspace(case)
        if case["op"].startswith("adapter"):
            s.adapters = s.work.adapters(s.a.data_ptr(), s.b.data_ptr(), s.scale.data_ptr(), GGUF[case["dtype"]], slots, r, k, n)
        else:
            s.config = s.work.router(e, top, case["norm"])
    return s


# ---- plain forms: elementary torch operations in 32 bits -------------------------------------------------------------------


def chosen(s):
    """[tokens, slots]: the scale of a token's adapter in the column of its slot, zero elsewhere."""
    one = (s.slot[:, None] == torch.arange(s.case["slots"], device="cuda")[None, :]).float()
    return one * s.scale[None, :]


def plain_adapter_forward(s):
    c = s.case
    a = s.a.float().reshape(-1, c["k"])                                             # [slots * rank, k]
    b = s.b.float().permute(0, 2, 1).reshape(-1, c["n"])                            # [slots * rank, n]
    h = (s.x @ a.T).view(c["tokens"], c["slots"], c["rank"]) * chosen(s)[:, :, None]
    return {"y": s.base + h.view(c["tokens"], -1) @ b}


def plain_adapter_backward(s):
    c = s.case
    t, slots, r = c["tokens"], c["slots"], c["rank"]
    a = s.a.float().reshape(-1, c["k"])
    b = s.b.float().permute(0, 2, 1).reshape(-1, c["n"])
    pick = chosen(s)[:, :, None]
    h = ((s.x @ a.T).view(t, slots, r) * pick).view(t, -1)
    g = ((s.dy @ b.T).view(t, slots, r) * pick).view(t, -1)
    db = (s.dy.T @ h).view(c["n"], slots, r).permute(1, 0, 2).contiguous()
    return {"dx": s.base + g @ a, "da": (g.T @ s.x).view(slots, r, c["k"]), "db": db}


def probabilities(s):
    """softmax of the logits, zero in the rows of padding, and the mask."""
    valid = torch.ones(s.case["tokens"], device="cuda", dtype=torch.bool) if s.mask is None else s.mask.bool()
    z = torch.where(valid[:, None], s.logits, torch.zeros_like(s.logits))
    e = torch.exp(z - z.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True) * valid[:, None], valid


def plain_balance_forward(s):
    e = s.case["experts"]
    p, valid = probabilities(s)
    at = torch.where(valid[:, None], s.ids.long(), torch.full_like(s.ids, e, dtype=torch.long)).reshape(-1)
    counts = torch.zeros(e + 1, device="cuda", dtype=torch.int32).scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    total = valid.sum().to(torch.int32)
    counts[e] = total
    sums = p.sum(0)
    n = total.float()
    return {"counts": counts, "prob_sums": sums, "loss": ((counts[:e].float() / n) * (sums / n)).sum()[None] * e}


def plain_balance_backward(s):
    c = s.case
    e = c["experts"]
    p, valid = probabilities(s)
    n = s.counts[e].float()
    f = s.counts[:e].float() * (s.loss_grad * e / (n * n))
    grad = p * (f[None, :] - (p * f[None, :]).sum(1, keepdim=True))
    chosen_p = p.gather(1, s.ids.long())
    dw = torch.where(valid[:, None], s.weights_grad, torch.zeros_like(s.weights_grad))
    if c["norm"]:
        z = torch.where(valid[:, None], s.logits.gather(1, s.ids.long()), torch.zeros_like(dw))
        w = torch.exp(z - z.amax(1, keepdim=True))
        w = w / w.sum(1, keepdim=True)
        return {"grad": grad.scatter_add_(1, s.ids.long(), w * (dw - (w * dw).sum(1, keepdim=True)))}
    grad = grad - p * (chosen_p * dw).sum(1, keepdim=True)
    return {"grad": grad.scatter_add_(1, s.ids.long(), chosen_p * dw)}


PLAIN = {"adapter forward": plain_adapter_forward, "adapter backward": plain_adapter_backward,
         "balance forward": plain_balance_forward, "balance backward": plain_balance_backward}


def run(s):
    if not own:
        return PLAIN[s.case["op"]](s)
    c, o = s.case, s.out
    if c["op"] == "adapter forward":
        s.work.adapter_forward(s.adapters, s.x.data_ptr(), s.slot.data_ptr(), s.base.data_ptr(), o["y"].data_ptr(), c["tokens"])
    elif c["op"] == "adapter backward":
        s.work.adapter_backward(s.adapters, s.x.data_ptr(), s.slot.data_ptr(), s.dy.data_ptr(), s.base.data_ptr(), o["dx"].data_ptr(),
                                o["da"].data_ptr(), o["db"].data_ptr(), c["tokens"])
    elif c["op"] == "balance forward":
        s.work.balance_forward(s.config, s.logits.data_ptr(), s.ids.data_ptr(), s.mask.data_ptr() if s.mask is not None else None, c["tokens"],
                               o["counts"].data_ptr(), o["prob_sums"].data_ptr(), o["loss"].data_ptr())
    else:
        s.work.balance_backward(s.config, s.logits.data_ptr(), s.ids.data_ptr(), s.mask.data_ptr() if s.mask is not None else None, c["tokens"],
                                s.counts.data_ptr(), s.loss_grad, s.weights_grad.data_ptr(), o["grad"].data_ptr())
    return o


def work(case):
    t = case["tokens"]
    if case["op"].startswith("adapter"):
        k, n, r, slots = case["k"], case["n"], case["rank"], case["slots"]
        used = slots * (1.0 - (1.0 - 1.0 / slots) ** case["requests"])              # expected number of adapters in use
        weights = used * r * (k + n) * (4 if case["dtype"] == "F32" else 2)
        if case["op"] == "adapter forward":
            return {"bytes": 4.0 * t * (k + 2 * n + 1) + weights, "flops": 2.0 * t * r * (k + n)}
        return {"bytes": 4.0 * t * (3 * k + n + 1) + weights + 4.0 * slots * r * (k + n), "flops": 2.0 * t * r * (3 * k + 2 * n)}
    e, top = case["experts"], case["top_k"]
    if case["op"] == "balance forward":
        return {"bytes": 4.0 * t * (e + top) + t + 8.0 * e, "flops": 6.0 * t * e}
    return {"bytes": 4.0 * t * (2 * e + 2 * top) + t + 4.0 * e, "flops": 10.0 * t * e}


def exact(case, seed):
    """The definitions, token groups and rows taken one by one, in 64 bits."""
    s = prepare(case, seed)
    t = case["tokens"]
    if case["op"].startswith("adapter"):
        x, a, b, scale = s.x.double(), s.a.double(), s.b.double(), s.scale.double()
        out = s.base.double().clone()
        if case["op"] == "adapter forward":
            for slot in range(case["slots"]):
                at = torch.nonzero(s.slot == slot).flatten()
                out[at] += scale[slot] * ((x[at] @ a[slot].T) @ b[slot].T)
            return {"y": out}
        dy, da, db = s.dy.double(), torch.zeros_like(a), torch.zeros_like(b)
        for slot in range(case["slots"]):
            at = torch.nonzero(s.slot == slot).flatten()
            g = scale[slot] * (dy[at] @ b[slot])
            out[at] += g @ a[slot]
            da[slot] = g.T @ x[at]
            db[slot] = scale[slot] * (dy[at].T @ (x[at] @ a[slot].T))
        return {"dx": out, "da": da, "db": db}
    e = case["experts"]
    rows = torch.arange(t, device="cuda") if s.mask is None else torch.nonzero(s.mask).flatten()
    n = rows.numel()
    z, ids = s.logits[rows].double(), s.ids[rows].long()
    log_p = z - torch.logsumexp(z, 1, keepdim=True)
    p = log_p.exp()
    hit = torch.zeros(n, e, device="cuda", dtype=torch.bool).scatter_(1, ids, True)
    counts = hit.sum(0)
    if case["op"] == "balance forward":
        share = counts.double() / n
        return {"counts": torch.cat([counts, torch.tensor([n], device="cuda")]).to(torch.int32), "prob_sums": p.sum(0),
                "loss": e * (share * p.mean(0)).sum()[None]}
    # d loss / d p, then the softmax's Jacobian; the route weights' likewise, through the chosen logits
    dp = (s.loss_grad * e / n / n) * counts.double()[None, :].expand(n, e).clone()
    dw = s.weights_grad[rows].double()
    grad = torch.zeros(t, e, device="cuda", dtype=torch.float64)
    if case["norm"]:
        w = log_p.gather(1, ids).softmax(1)
        through = torch.zeros(n, e, device="cuda", dtype=torch.float64).scatter_(1, ids, w * dw - w * (w * dw).sum(1, keepdim=True))
    else:
        dp.scatter_add_(1, ids, dw)
        through = 0.0
    grad[rows] = p * dp - p * (p * dp).sum(1, keepdim=True) + through
    return {"grad": grad}
