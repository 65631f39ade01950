"""Cases of the gradient norm, the clipping by it and the weight update that follows a physics loss's backward pass.

A training step hands over one gradient for every parameter tensor: a few dozen small ones where only low-rank adapters
are trained, a few hundred of all sizes where the whole network is.  Here the tensors of a case lie in one buffer, one
behind the other (`packed`: without any padding, as buckets of a data-parallel run hold them, so that odd sizes leave
the next tensor unaligned; otherwise each on a 256-byte border, as separate allocations are).  The plain forms work on
the whole buffer, the framework's calls on the list of tensors.
"""
import math

import torch

own = False

LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01


def listed():
    return [
        # latency: the adapters (rank 8) of a small 4-block network, 48 tensors of 2 k to 8 k values
        dict(name="norm_adapters", op="norm", layout="adapters", blocks=4, width=256, rank=8, packed=False, dtype="float32", norm="2", each=False),
        # largest magnitude of the gradients of an odd-width convolution network, logged each step
        dict(name="norm_convs_inf", op="norm", layout="convs", blocks=20, width=61, rank=0, packed=True, dtype="float16", norm="inf", each=False),
        # total and per-tensor norms, logged per layer, of a 12-block network in bfloat16
        dict(name="norm_each_bf16", op="norm", layout="network", blocks=12, width=1024, rank=0, packed=False, dtype="bfloat16", norm="2", each=True),
        # the whole gradient of the largest network, float32
        dict(name="norm_largest", op="norm", layout="network", blocks=24, width=1536, rank=0, packed=False, dtype="float32", norm="2", each=False),
        # adapters (rank 16) of a 12-block network: the usual fine-tuning step, 144 tensors
        dict(name="clip_adapters", op="clip", layout="adapters", blocks=12, width=512, rank=16, packed=False, dtype="float32", clips=True),
        # odd sizes, unpadded bfloat16: every second tensor starts off any 4-byte border
        dict(name="clip_convs_odd", op="clip", layout="convs", blocks=24, width=173, rank=0, packed=True, dtype="bfloat16", clips=True),
        # whole network, float32: more than the on-chip caches hold
        dict(name="clip_network", op="clip", layout="network", blocks=12, width=1024, rank=0, packed=False, dtype="float32", clips=True),
        # first step of the smallest fine-tuning
        dict(name="adamw_adapters", op="adamw", layout="adapters", blocks=4, width=256, rank=8, packed=False, dtype="float32", clips=True, steps=0),
        # convolution network without clipping, odd sizes without padding
        dict(name="adamw_convs_odd", op="adamw", layout="convs", blocks=24, width=173, rank=0, packed=True, dtype="float32", clips=False, steps=1000),
        # bfloat16 network with 32-bit master weights
        dict(name="adamw_bf16", op="adamw", layout="network", blocks=12, width=1024, rank=0, packed=False, dtype="bfloat16", clips=True, steps=200),
        # whole network in float32, the largest step
        dict(name="adamw_largest", op="adamw", layout="network", blocks=16, width=1536, rank=0, packed=False, dtype="float32", clips=True, steps=1000),
    ]


def draw(rng):
    op = rng.choice(["norm", "clip", "adamw"])
    layout = rng.choice(["adapters", "network", "convs"])
    high = {"adapters": 2048, "network": 1024, "convs": 512}[layout]
    case = dict(op=op, layout=layout, blocks=rng.randint(1, 12), width=int(round(math.exp(rng.uniform(math.log(17), math.log(high))))),
                rank=rng.choice([1, 4, 5, 8, 16, 32]), packed=rng.random() < 0.5,
                dtype=rng.choice(["float32", "bfloat16"] if op == "adamw" else ["float32", "bfloat16", "float16"]))
    if op == "norm":
        case.update(norm=rng.choice(["1", "2", "2", "inf"]))
        case.update(each=case["norm"] != "inf" and rng.random() < 0.5)
    else:
        case.update(clips=rng.random() < 0.75)
    if op == "adamw":
        case.update(steps=rng.choice([0, 1, 30, 1000, 20000]))
    return case


def _sizes(case):
    w, r = case["width"], case["rank"]
    if case["layout"] == "adapters":      # two factors for each of the four w x w and the two w x 4w products of a block
        block = [r * w] * 8 + [r * w, r * 4 * w] * 2
    elif case["layout"] == "network":     # weights and biases of those products, two norms
        block = [w * w, w] * 4 + [4 * w * w, 4 * w, 4 * w * w, w] + [w] * 4
    else:                                 # a 3 x 3 convolution with bias, and a scale
        block = [9 * w * w, w, w]
    return block * case["blocks"]


def _inputs(case, seed):
    """The step's tensors: one buffer of each kind, zero between the tensors, and the tensors as views of it."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, sizes, at, places = getattr(torch, case["dtype"]), _sizes(case), 0, []
    for n in sizes:
        places.append((at, at + n))
        at += n if case["packed"] else -(-n // 128) * 128
    scales = torch.rand(len(sizes), generator=gen, device="cuda").mul(4).sub(4).mul(math.log(10)).exp().tolist()      # 1e-4 .. 1 by tensor

    def values(dtype, make):
        flat = torch.zeros(at, dtype=dtype, device="cuda")
        for (a, b), s in zip(places, scales):
            make(flat[a:b], s)
        return flat, [flat[a:b] for a, b in places]

    state = dict(case=case, places=places)
    state["grad"], state["grads"] = values(dtype, lambda x, s: x.normal_(0.0, s, generator=gen))
    if case["op"] != "norm":
        size = float(torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt())
        state["max_norm"] = (0.3 if case["clips"] else 3.0) * size
    if case["op"] == "adamw":
        started = case["steps"] > 0
        wide, wides = values(torch.float32, lambda x, s: x.normal_(0.0, 0.05, generator=gen))
        state["exp_avg"], state["exp_avgs"] = values(torch.float32, lambda x, s: x.normal_(0.0, 0.1 * s, generator=gen) if started else x)
        state["exp_avg_sq"], state["exp_avg_sqs"] = values(torch.float32, lambda x, s: x.normal_(0.0, s, generator=gen).square_() if started else x)
        state["steps"] = torch.full((len(sizes),), float(case["steps"]), device="cuda")
        if dtype == torch.float32:
            state["param"] = wide
        else:
            state["master"], state["masters"], state["param"] = wide, wides, wide.to(dtype)
    elif case["op"] == "clip":
        state["param"] = torch.zeros_like(state["grad"])
    if "param" in state:
        state["params"] = [state["param"][a:b] for a, b in places]
        for p, g in zip(state["params"], state["grads"]):
            p.requires_grad_(True).grad = g
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["op"] == "adamw":      # the optimizer object that a training program builds once
        import pde_amd
        opt = pde_amd.ClippedAdamW(state["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                   max_norm=state["max_norm"] if case["clips"] else None)
        for i, p in enumerate(state["params"]):      # the state of a resumed run
            opt.state[p] = dict(step=state["steps"][i], exp_avg=state["exp_avgs"][i], exp_avg_sq=state["exp_avg_sqs"][i])
            if "masters" in state:
                opt.state[p]["master"] = state["masters"][i]
        state["optimizer"] = opt
    return state


def _total(x, norm):
    return x.abs().amax() if norm == "inf" else x.abs().sum() if norm == "1" else x.square().sum().sqrt()


def _norm(state):
    case = state["case"]
    x = state["grad"].float()
    total = _total(x, case["norm"])
    if not case["each"]:
        return total
    # sums of neighbouring stretches, from one running sum in 64 bits
    running = torch.cumsum((x.abs() if case["norm"] == "1" else x.square()).double(), 0)
    ends = torch.tensor([b - 1 for _, b in state["places"]], device=x.device)
    parts = torch.diff(running[ends], prepend=running.new_zeros(1))
    return total, (parts if case["norm"] == "1" else parts.sqrt()).float()


def _coefficient(x, max_norm):
    total = _total(x, "2")
    return total, (max_norm / (total + 1e-6)).clamp(max=1.0)


def _clip(state):
    x = state["grad"].float()
    total, c = _coefficient(x, state["max_norm"])
    state["grad"].copy_(x * c)
    return total, state["grad"]


def _adamw(state):
    x, w = state["grad"].float(), state.get("master", state["param"].detach())
    if state["case"]["clips"]:
        x = x * _coefficient(x, state["max_norm"])[1]
    m, v = state["exp_avg"], state["exp_avg_sq"]
    t = state["steps"].add_(1)[0].double()
    bias1, bias2 = (1 - BETA1 ** t).float(), (1 - BETA2 ** t).float()
    m.mul_(BETA1).add_(x, alpha=1 - BETA1)
    v.mul_(BETA2).add_(x * x, alpha=1 - BETA2)
    w.mul_(1 - LR * DECAY).sub_(m / (v.sqrt() / bias2.sqrt() + EPS) * (LR / bias1))
    if "master" in state:
        state["param"].detach().copy_(w)
    return _updated(state)


def _updated(state):
    return [state[k].detach() for k in ("param", "exp_avg", "exp_avg_sq", "steps", "master") if k in state]


def run(state):
    case = state["case"]
    if case["op"] == "clip" and case["clips"]:
        state["max_norm"] *= 0.9999      # a threshold that falls step by step, so that each pass has something to clip
    if not own:
        return {"norm": _norm, "clip": _clip, "adamw": _adamw}[case["op"]](state)
    import pde_amd
    if case["op"] == "norm":
        return pde_amd.get_total_norm(state["grads"], float(case["norm"]), per_tensor=case["each"])
    if case["op"] == "clip":
        return pde_amd.clip_grad_norm_(state["params"], state["max_norm"]), state["grad"]
    state["optimizer"].step()
    return _updated(state)


def exact(case, seed):
    state = _inputs(case, seed)
    x = state["grad"].double()
    if case["op"] == "norm":
        p = float(case["norm"])
        total = torch.linalg.vector_norm(x, p)
        return (total, torch.stack([torch.linalg.vector_norm(x[a:b], p) for a, b in state["places"]])) if case["each"] else total
    total = torch.dot(x, x) ** 0.5
    scale = 1.0
    if case["clips"] or case["op"] == "clip":
        limit = state["max_norm"] * (0.9999 if case["op"] == "clip" and case["clips"] else 1.0)
        scale = min(1.0, limit / (float(total) + 1e-6))
    x *= scale
    if case["op"] == "clip":
        return total, x
    n = case["steps"] + 1
    w = state.get("master", state["param"].detach()).double()
    m = torch.lerp(x, state["exp_avg"].double(), BETA1)
    v = torch.lerp(x.square_(), state["exp_avg_sq"].double(), BETA2)
    step = (m / (1 - BETA1 ** n)) / ((v / (1 - BETA2 ** n)).sqrt_().add_(EPS))
    w -= LR * (step + DECAY * w)
    out = [w, m, v, torch.full((len(state["places"]),), float(n), dtype=torch.float64)]
    return out + [w] if "master" in state else out


def work(case):
    n = sum(_sizes(case))
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        return dict(bytes=n * e + (4 * len(_sizes(case)) if case["each"] else 0), flops=2 * n)
    if case["op"] == "clip":
        return dict(bytes=2 * n * e, flops=3 * n)
    # reads gradient, weight and both moments, writes the latter three, and the rounded weight where it has fewer bits
    return dict(bytes=n * (e + 12 + 12 + (e if e < 4 else 0)), flops=14 * n)
