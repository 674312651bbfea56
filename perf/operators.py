"""Operators of a sequence policy as measurable cases: a recurrent memory of
linear attention with a decay for each head (chunked over a sequence, forward
and backward; one token at a time when acting), the gated projections of a
feed-forward block (forward and backward), and the AdamW step over many
tensors with its moments in 32 or in 8 bits.

With `own` false `run` computes them in plain torch operations, with `own`
true through the package's public entry points: training passes as captured
train steps, as this package runs its updates, single tokens and rows as a
captured trace, as its acting nets run, prompts and optimizer steps as eager
calls.  `exact` computes the same in float64, step by step.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tt-rl_amd"))

own = False

CHUNK = 64  # steps of the plain form's chunks
BLOCK = 64  # elements that share a scale where moments are held in 8 bits
BETA1, BETA2, EPS, LR, DECAY, STEPS_DONE = 0.9, 0.999, 1e-8, 3e-4, 0.01, 10


# ------------------------------------------------------------------ cases ---

def listed() -> list:
    return [
        # one environment acting: a single token through the memory of a policy of width 512
        {"name": "token_1", "kind": "token", "lanes": 1, "heads": 8, "kv_heads": 8, "key": 64, "value": 64,
         "decay": "head", "done": True},
        # a large vector environment, the states of 1000 lanes read and written once
        {"name": "token_1000", "kind": "token", "lanes": 1000, "heads": 8, "kv_heads": 4, "key": 64, "value": 64,
         "decay": "step", "done": True},
        # the recurrent PPO minibatch of this repository: 16 sequences of 32 steps with episode resets
        {"name": "memory_32x16", "kind": "memory", "steps": 32, "batch": 16, "heads": 8, "kv_heads": 8, "key": 64,
         "value": 64, "decay": "head", "done": True, "final_grad": False},
        # long episodes in a large batch: many rows, the memory's traffic
        {"name": "memory_1024x32", "kind": "memory", "steps": 1024, "batch": 32, "heads": 8, "kv_heads": 8, "key": 64,
         "value": 64, "decay": "head", "done": True, "final_grad": False},
        # few rows and a long axis, odd widths, shared key/value heads, a decay for each step
        {"name": "memory_4001x2", "kind": "memory", "steps": 4001, "batch": 2, "heads": 6, "kv_heads": 3, "key": 40,
         "value": 72, "decay": "step", "done": True, "final_grad": True},
        # a prompt run into a state without gradients: heads of 128
        {"name": "prompt_2048x8", "kind": "prompt", "steps": 2048, "batch": 8, "heads": 8, "kv_heads": 8, "key": 128,
         "value": 128, "decay": "step", "done": False},
        # one observation through the gated projections: the weights' traffic
        {"name": "gated_1", "kind": "gated_act", "rows": 1, "in": 512, "hidden": 2048, "act": "silu", "bias": False},
        # ragged rows and widths, biases
        {"name": "gated_777", "kind": "gated", "rows": 777, "in": 500, "hidden": 1333, "act": "gelu", "bias": True},
        # a training batch of a large policy: the matrix cores
        {"name": "gated_8192", "kind": "gated", "rows": 8192, "in": 1024, "hidden": 4096, "act": "silu", "bias": False},
        # the Nature-CNN Q network's ten tensors, moments in 32 bits
        {"name": "adamw_cnn", "kind": "adamw", "bits": 32, "set": "cnn", "width": 512, "layers": 1},
        # four blocks of a sequence policy, twenty tensors, moments in 8 bits
        {"name": "adamw8_1024", "kind": "adamw", "bits": 8, "set": "block", "width": 1024, "layers": 4},
        # tensors of odd sizes, moments in 8 bits
        {"name": "adamw8_odd", "kind": "adamw", "bits": 8, "set": "odd", "width": 201, "layers": 4},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["token", "memory", "memory", "prompt", "gated_act", "gated", "gated", "adamw"])
    if kind in ("token", "memory", "prompt"):
        share = rng.choice([1, 1, 2, 4])
        kv = rng.choice([1, 2, 3, 4, 8])
        c = {"kind": kind, "heads": kv * share, "kv_heads": kv, "key": rng.choice([16, 32, 48, 64, 64, 96, 128, rng.randint(8, 128)]),
             "value": rng.choice([16, 32, 64, 64, 96, 128, rng.randint(8, 128)]), "decay": rng.choice(["head", "step"]),
             "done": rng.random() < 0.6}
        wide = max(c["key"], c["value"])
        if kind == "token":
            c["lanes"] = _log_int(rng, 1, max(1, min(4096, (1 << 25) // (c["heads"] * c["key"] * c["value"]))))
            return c
        rows = (1 << 24) // (c["heads"] * wide)  # elements of the widest operand at most
        c["steps"] = _log_int(rng, 1, min(rows, 8000))
        c["batch"] = _log_int(rng, 1, max(1, min(256, rows // c["steps"])))
        if kind == "memory":
            c["final_grad"] = rng.random() < 0.3
        return c
    if kind in ("gated_act", "gated"):
        c = {"kind": kind, "in": rng.choice([64, 128, 256, 500, 512, 777, 1024, rng.randint(8, 1024)]),
             "hidden": rng.choice([128, 256, 512, 1024, 1333, 2048, 4096, rng.randint(8, 4096)]),
             "act": rng.choice(["silu", "gelu", "relu", "sigmoid"]), "bias": rng.random() < 0.5}
        c["rows"] = _log_int(rng, 1, 64 if kind == "gated_act" else 8192)
        return c
    return {"kind": kind, "bits": rng.choice([8, 8, 32]), "set": rng.choice(["cnn", "block", "odd"]),
            "width": _log_int(rng, 64, 1024), "layers": rng.randint(1, 4)}


# ----------------------------------------------------------------- inputs ---

def _rng(seed: int):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _uniform(gen, bound: float, *shape):
    return (torch.rand(shape, generator=gen, device="cuda") * 2 - 1) * bound


def _memory_inputs(c, seed):
    gen = _rng(seed)
    T, B = (1, c["lanes"]) if c["kind"] == "token" else (c["steps"], c["batch"])
    H, G, K, V = c["heads"], c["kv_heads"], c["key"], c["value"]
    t = {"q": _normal(gen, T, B, H, K), "k": F.normalize(_normal(gen, T, B, G, K), dim=-1), "v": _normal(gen, T, B, G, V)}
    # a head keeps between 3/4 and 1 - 1/256 of its state over a step, or what its own gate says
    keep = 1.0 - torch.exp2(-2.0 - 6.0 * torch.arange(H, device="cuda") / max(1, H - 1))
    head = torch.log(keep).reshape(1, H)
    t["log_decay"] = head if c["decay"] == "head" else F.logsigmoid(_normal(gen, T, B, H) + 2.5)
    t["state"] = 0.5 * _normal(gen, B, H, K, V)
    t["done"] = (torch.rand((T, B, 1), generator=gen, device="cuda") < 0.01).float() if c["done"] else None
    if c["kind"] == "memory":
        t["dout"] = _normal(gen, T, B, H, V)
        t["dfinal"] = _normal(gen, B, H, K, V) if c["final_grad"] else None
    if c["kind"] == "token":
        for name in ("q", "k", "v", "done"):
            t[name] = None if t[name] is None else t[name][0]
        if c["decay"] == "step":
            t["log_decay"] = t["log_decay"][0]
    return t


def _gated_inputs(c, seed):
    gen, bound = _rng(seed), 1.0 / math.sqrt(c["in"])
    t = {"x": _normal(gen, c["rows"], c["in"])}
    t["w_gate"], t["w_up"] = (_uniform(gen, bound, c["in"], c["hidden"]) for _ in range(2))
    t["b_gate"], t["b_up"] = ((_uniform(gen, bound, 1, c["hidden"]) if c["bias"] else None) for _ in range(2))
    if c["kind"] == "gated":
        t["dout"] = _normal(gen, c["rows"], c["hidden"])
        if c["act"] == "relu":
            # Relu's slope has no value where rounding decides the gate's sign: nothing is asked of such elements.
            g = t["x"].double() @ t["w_gate"].double()
            g = g if t["b_gate"] is None else g + t["b_gate"].double()
            t["dout"].masked_fill_(g.abs() < 1e-4, 0.0)
    return t


def _shapes(c) -> list:
    w = c["width"]
    if c["set"] == "cnn":
        return [(256, 32), (1, 32), (512, 64), (1, 64), (576, 64), (1, 64), (3136, w), (1, w), (w, 6), (1, 6)]
    if c["set"] == "block":
        return [s for _ in range(c["layers"]) for s in ((w, 3 * w), (w, w), (w, 4 * w), (w, 4 * w), (4 * w, w))]
    return [(w + 7 * i + 1, w + 5 * j) for i in range(c["layers"]) for j in (0, 3)] + [(1, w + i) for i in range(c["layers"])]


def _count(shape) -> int:
    return shape[0] * shape[1]


def _places(shapes) -> list:
    """Where each tensor starts in a buffer whose tensors start on blocks."""
    at, out = 0, []
    for s in shapes:
        out.append(at)
        at += -(-_count(s) // BLOCK) * BLOCK
    return out + [at]


def _adamw_inputs(c, seed):
    gen, shapes = _rng(seed), _shapes(c)
    places = _places(shapes)
    real = torch.zeros(places[-1], dtype=torch.bool, device="cuda")
    for s, at in zip(shapes, places):
        real[at:at + _count(s)] = True
    n = places[-1]
    flat = {"p": 0.05 * _normal(gen, n), "g": 0.01 * _normal(gen, n) * torch.exp(_normal(gen, n)),
            "m": 0.003 * _normal(gen, n), "v": (0.01 * _normal(gen, n)).square()}
    flat = {k: torch.where(real, a, torch.zeros_like(a)) for k, a in flat.items()}
    if c["bits"] == 8:
        for name, fn in (("m", _hold_m), ("v", _hold_v)):
            flat[name + "_codes"], flat[name + "_scale"] = fn(flat.pop(name))
    return {"flat": flat, "shapes": shapes, "places": places}


# -------------------------------------------------------------- plain forms ---

def _sums(g):
    """[..., i, j] = g[j + 1] + ... + g[i] for j <= i, else -inf; each row of
    sums starts at its own j, so that near steps lose nothing to far ones."""
    n = g.shape[-1]
    i = torch.arange(n, device=g.device)
    terms = g.unsqueeze(-1).expand(*g.shape, n).masked_fill(i[:, None] <= i[None, :], 0.0)
    return terms.cumsum(-2).masked_fill(i[:, None] < i[None, :], -math.inf)


def _plain_memory(q, k, v, log_decay, state, done):
    """Chunks of CHUNK steps: products inside a chunk, and the chunks' states
    joined by the decays between them."""
    T, B, H, K = q.shape
    V = v.shape[-1]
    g = log_decay.expand(T, B, H) if log_decay.dim() == 2 else log_decay
    if done is not None:
        g = g.masked_fill(done > 0, -math.inf)
    rest = -T % CHUNK
    N = (T + rest) // CHUNK

    def chunks(x):  # (T, B, heads, n) -> (B, H, N, CHUNK, n)
        x = F.pad(x, (0, 0, 0, 0, 0, 0, 0, rest)).repeat_interleave(H // x.shape[2], dim=2)
        return x.reshape(N, CHUNK, B, H, -1).permute(2, 3, 0, 1, 4).contiguous()

    q, k, v = chunks(q), chunks(k), chunks(v)
    g = F.pad(g, (0, 0, 0, 0, 0, rest)).reshape(N, CHUNK, B, H).permute(2, 3, 0, 1).contiguous()
    within = torch.exp(_sums(g))
    into = torch.exp(g.cumsum(-1)).unsqueeze(-1)
    total = g.sum(-1)
    inside = torch.matmul(torch.matmul(q, k.transpose(-1, -2).contiguous()) * within, v)
    added = torch.matmul((k * within[..., -1, :].unsqueeze(-1)).transpose(-1, -2).contiguous(), v)
    parts = torch.cat([state.unsqueeze(2), added], 2).reshape(B, H, N + 1, K * V)
    states = torch.matmul(torch.exp(_sums(F.pad(total, (1, 0)))), parts).reshape(B, H, N + 1, K, V)
    out = (inside + into * torch.matmul(q, states[:, :, :N])) * (1.0 / math.sqrt(K))
    out = out.permute(2, 3, 0, 1, 4).reshape(N * CHUNK, B, H, V)[:T]
    return out, states[:, :, N]


def _plain_memory_grads(t):
    names = ("q", "k", "v", "log_decay", "state")
    leaves = {n: t[n].detach().requires_grad_() for n in names}
    out, final = _plain_memory(*(leaves[n] for n in names), t["done"])
    outs, douts = ((out, final), (t["dout"], t["dfinal"])) if t["dfinal"] is not None else ((out,), (t["dout"],))
    grads = torch.autograd.grad(outs, list(leaves.values()), douts)
    return {"out": out.detach(), "final": final.detach(), "grads": dict(zip(names, grads))}


def _plain_token(t):
    q, k, v, S = t["q"], t["k"], t["v"], t["state"]
    share = q.shape[1] // k.shape[1]
    keep = torch.exp(t["log_decay"])[..., None, None]
    if t["done"] is not None:
        keep = keep * (t["done"] <= 0)[..., None, None]
    k, v = (x.repeat_interleave(share, dim=1) for x in (k, v))
    S.mul_(keep).add_(k.unsqueeze(-1) * v.unsqueeze(-2))
    return {"out": (q.unsqueeze(-1) * S).sum(-2) * (1.0 / math.sqrt(q.shape[-1])), "state": S}


def _gate(act: str, g):
    """The activation and its derivative."""
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "gelu":
        half = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * half, half + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-g))
    return (s, s * (1.0 - s)) if act == "sigmoid" else (g * s, s * (1.0 + g * (1.0 - s)))


def _projections(t):
    g, u = t["x"] @ t["w_gate"], t["x"] @ t["w_up"]
    return (g, u) if t["b_gate"] is None else (g + t["b_gate"], u + t["b_up"])


def _plain_gated(t, act):
    g, u = _projections(t)
    return {"out": _gate(act, g)[0] * u}


def _plain_gated_grads(t, act):
    g, u = _projections(t)
    a, slope = _gate(act, g)
    du, dg = t["dout"] * a, t["dout"] * u * slope
    xt = t["x"].T
    grads = {"x": dg @ t["w_gate"].T + du @ t["w_up"].T, "w_gate": xt @ dg, "w_up": xt @ du}
    if t["b_gate"] is not None:
        grads.update(b_gate=dg.sum(0, keepdim=True), b_up=du.sum(0, keepdim=True))
    return {"out": a * u, "grads": grads}


def _ratio(a):
    """|a| over its block's largest, and that largest."""
    a = a.reshape(-1, BLOCK).abs()
    top = a.amax(1, keepdim=True)
    return torch.where(top > 0, a / top, torch.zeros_like(a)), top


def _hold_m(m):
    """127 signed steps of the square root: code c stands for (c / 127)^2 of its block's largest."""
    r, top = _ratio(m)
    codes = torch.round(torch.sqrt(r) * 127.0) * torch.sign(m.reshape(-1, BLOCK))
    return codes.to(torch.int8).reshape(-1), top.reshape(-1)


def _held_m(codes, scale):
    c = codes.reshape(-1, BLOCK).float() * (1.0 / 127.0)
    return (c * c.abs() * scale.reshape(-1, 1)).reshape(-1)


def _hold_v(v):
    """255 steps of the fourth root; what is not zero is never held as zero."""
    r, top = _ratio(v)
    codes = torch.round(torch.sqrt(torch.sqrt(r)) * 255.0)
    codes = torch.where(r > 0, codes.clamp(min=1.0), codes)
    return codes.to(torch.uint8).reshape(-1), top.reshape(-1)


def _held_v(codes, scale):
    c = codes.reshape(-1, BLOCK).float() * (1.0 / 255.0)
    c = c * c
    return (c * c * scale.reshape(-1, 1)).reshape(-1)


def _plain_adamw(state, bits):
    """One pass over all tensors, laid end to end; every product and sum is rounded on its own."""
    f = state["flat"]
    state["t"] += 1
    bc1, bc2 = 1.0 - BETA1 ** state["t"], 1.0 - BETA2 ** state["t"]
    m, v = (f["m"], f["v"]) if bits == 32 else (_held_m(f["m_codes"], f["m_scale"]), _held_v(f["v_codes"], f["v_scale"]))
    g = f["g"]
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    step = m / (torch.sqrt(v) * (1.0 / math.sqrt(bc2)) + EPS) * (LR / bc1)
    f["p"].copy_(f["p"] * (1.0 - LR * DECAY) - step)
    if bits == 32:
        f["m"].copy_(m)
        f["v"].copy_(v)
    else:
        for name, a, hold, held in (("m", m, _hold_m, _held_m), ("v", v, _hold_v, _held_v)):
            codes, scale = hold(a)
            f[name + "_codes"].copy_(codes)
            f[name + "_scale"].copy_(scale)
        m, v = _held_m(f["m_codes"], f["m_scale"]), _held_v(f["v_codes"], f["v_scale"])
    return {"p": _split(f["p"], state), "m": _split(m, state), "v": _split(v, state)}


def _split(flat, state) -> list:
    return [flat[at:at + _count(s)].view(s) for s, at in zip(state["shapes"], state["places"])]


# ------------------------------------------------------------- the package ---

def _device():
    from ttrl_amd.engine.device import open_device

    return open_device(0)


class _Memory:
    """A device array of the package, as torch sees foreign device memory."""

    def __init__(self, array):
        self.array = array
        self.__cuda_array_interface__ = {"shape": tuple(array.shape), "typestr": array.dtype.str,
                                         "data": (array.ptr, False), "version": 2, "strides": None}


def _see(x):
    return torch.as_tensor(_Memory(getattr(x, "data", x)), device="cuda")


def _tensors(t, grad=()) -> dict:
    """The package's tensors with the values of torch's."""
    import ctypes

    from ttrl_amd.engine.autograd import Tensor
    from ttrl_amd.engine.tensor import DeviceArray

    dev, out = _device(), {}
    torch.cuda.synchronize()
    for name, a in t.items():
        if a is None:
            continue
        a = a.contiguous()
        d = DeviceArray(dev, a.shape)
        dev.call("ttrl_d2d", d.vp, ctypes.c_void_p(a.data_ptr()), ctypes.c_size_t(d.nbytes))
        dev.synchronize()
        out[name] = Tensor(d, name in grad)
    return out


def _train_step(inputs, leaves, forward):
    """A captured forward and backward of what `forward` returns, and its outputs as torch sees them."""
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.step import TrainStep

    made = {}

    def body(x):
        for t in x.values():
            t.zero_grad()
        made["outs"], seeds = forward(x)
        backward_from(seeds)
        return {}

    step = TrainStep(body, inputs, _device(), mode="graph")
    step.run()
    out = {n: _see(o) for n, o in made["outs"].items()}
    out["grads"] = {n: _see(inputs[n].grad) for n in leaves if n in inputs}
    return {"step": step, "made": made, "out": out}


def _trace(record):
    """A captured call, replayed as single launches as the acting nets do."""
    from ttrl_amd.engine.autograd import no_grad
    from ttrl_amd.engine.trace import capture

    def quiet():
        with no_grad():
            return record()

    dev = _device()
    pool = dev.create_pool()
    with dev.use_pool(pool):
        made = quiet()  # fills the pool
        del made
        dev.synchronize()
        trace, made = capture(dev, quiet)
    trace.set_direct()
    return {"trace": trace, "made": made}


def _own_memory(c, t):
    from ttrl_amd.engine.ops import linear_attention, linear_attention_step

    if c["kind"] == "memory":
        leaves = ("q", "k", "v", "log_decay", "state")
        x = _tensors(t, leaves)

        def forward(x):
            out, final = linear_attention(x["q"], x["k"], x["v"], x["log_decay"], x["state"], x.get("done"))
            seeds = [(out, x["dout"])] + ([(final, x["dfinal"])] if "dfinal" in x else [])
            return {"out": out, "final": final}, seeds

        return _train_step(x, leaves, forward)
    x = _tensors(t)
    if c["kind"] == "prompt":
        return {"x": x, "call": lambda: linear_attention(x["q"], x["k"], x["v"], x["log_decay"], x["state"], x.get("done"))}
    start = t["state"]
    s = _trace(lambda: linear_attention_step(x["q"], x["k"], x["v"], x["log_decay"], x["state"], x.get("done")))
    x["state"].data.copy_from(_tensors({"state": start})["state"].data)  # filling the pool was a step too
    s.update(x=x, out={"out": _see(s["made"]), "state": _see(x["state"])})
    return s


def _own_gated(c, t):
    from ttrl_amd.engine.ops import gated_linear

    leaves = ("x", "w_gate", "w_up", "b_gate", "b_up") if c["kind"] == "gated" else ()
    x = _tensors(t, leaves)

    def call(x=x):
        return gated_linear(x["x"], x["w_gate"], x["w_up"], x.get("b_gate"), x.get("b_up"), activation=c["act"])

    if c["kind"] == "gated":
        def forward(x):
            h = call(x)
            return {"out": h}, [(h, x["dout"])]

        return _train_step(x, leaves, forward)
    s = _trace(call)
    s.update(x=x, out={"out": _see(s["made"])})
    return s


def _own_adamw(c, state):
    from ttrl_amd.engine.optim import AdamW
    from ttrl_amd.engine.tensor import DeviceArray

    def each(flat):
        return _split(flat, state)

    f, n = state["flat"], len(state["shapes"])
    params = _tensors({i: p for i, p in enumerate(each(f["p"]))}, range(n))
    grads = _tensors({i: g for i, g in enumerate(each(f["g"]))})
    params = [params[i] for i in range(n)]
    for i, p in enumerate(params):
        p.grad = grads[i].data
    opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=c["bits"])
    saved = {"t": STEPS_DONE}
    for name in ("m", "v"):
        if c["bits"] == 32:
            saved[name] = [a.cpu().numpy() for a in each(f[name])]
        else:
            saved[name] = [a.cpu().numpy() for a in each(f[name + "_codes"])]
            scale = f[name + "_scale"].cpu().numpy()
            saved[name + "_scale"] = [scale[at // BLOCK:(at + _count(s) + BLOCK - 1) // BLOCK]
                                      for s, at in zip(state["shapes"], state["places"])]
    opt.load_state_dict(saved)
    held = None
    if c["bits"] == 8:
        held = tuple([DeviceArray(_device(), s) for s in state["shapes"]] for _ in range(2))
    m, v = held if held else (opt.m, opt.v)
    return {"opt": opt, "params": params, "grads": grads, "held": held,
            "out": {"p": [_see(p) for p in params], "m": [_see(a) for a in m], "v": [_see(a) for a in v]}}


# ---------------------------------------------------------------- the calls ---

def prepare(case: dict, seed: int):
    """Inputs from the seed; for the package, in its own memory, with the
    captured step or the optimizer that its user keeps."""
    kind = case["kind"]
    if kind == "adamw":
        t = _adamw_inputs(case, seed)
        t["t"] = STEPS_DONE
        mine = _own_adamw(case, t) if own else None
    elif kind in ("gated", "gated_act"):
        t = _gated_inputs(case, seed)
        mine = _own_gated(case, t) if own else None
    else:
        t = _memory_inputs(case, seed)
        mine = _own_memory(case, t) if own else None
    return {"case": case, "inputs": None if own else t, "own": mine}


def run(state):
    case, t, s = state["case"], state["inputs"], state["own"]
    kind = case["kind"]
    if own:
        if kind == "prompt":
            s["kept"] = s["call"]()
            out, final = s["kept"]
            return {"out": _see(out), "final": _see(final)}
        if kind == "adamw":
            s["opt"].step()
            if s["held"]:
                s["opt"].moments(out=s["held"])
            return s["out"]
        if "step" in s:
            s["step"].replay()
        else:
            s["trace"].replay()
        return s["out"]
    if kind == "adamw":
        return _plain_adamw(t, case["bits"])
    if kind == "gated":
        return _plain_gated_grads(t, case["act"])
    if kind == "gated_act":
        return _plain_gated(t, case["act"])
    if kind == "token":
        return _plain_token(t)
    if kind == "memory":
        return _plain_memory_grads(t)
    out, final = _plain_memory(t["q"], t["k"], t["v"], t["log_decay"], t["state"], t["done"])
    return {"out": out, "final": final}


# ---------------------------------------------------------- float64 twins ---

def _exact_memory(c, t):
    """S_t = a_t S_{t-1} + k_t v_t^T and o_t = q_t S_t / sqrt(K), step by step;
    the gradients from the same recurrence walked back."""
    d = {n: None if a is None else a.double() for n, a in t.items()}
    if c["kind"] == "token":
        d.update({n: d[n].unsqueeze(0) for n in ("q", "k", "v")}, done=None if d["done"] is None else d["done"].unsqueeze(0))
        if c["decay"] == "step":
            d["log_decay"] = d["log_decay"].unsqueeze(0)
    T, B, H, K = d["q"].shape
    share, scale = H // d["k"].shape[2], 1.0 / math.sqrt(K)
    q, k, v = d["q"] * scale, d["k"].repeat_interleave(share, 2), d["v"].repeat_interleave(share, 2)
    a = torch.exp(d["log_decay"]).expand(T, B, H).clone()
    if d["done"] is not None:
        a = a * (d["done"] <= 0)
    train = c["kind"] == "memory"
    S, states, outs = d["state"], [], []
    for i in range(T):
        if train:
            states.append(S)
        S = a[i][..., None, None] * S + k[i].unsqueeze(-1) * v[i].unsqueeze(-2)
        outs.append(torch.matmul(q[i].unsqueeze(-2), S).squeeze(-2))
    out = torch.stack(outs)
    if c["kind"] == "token":
        return {"out": out[0], "state": S}
    if not train:
        return {"out": out, "final": S}
    G = d["dfinal"] if d["dfinal"] is not None else torch.zeros_like(S)
    dq, dk, dv, da = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(a)
    for i in reversed(range(T)):
        do = d["dout"][i]
        now = a[i][..., None, None] * states[i] + k[i].unsqueeze(-1) * v[i].unsqueeze(-2)
        dq[i] = (now * do.unsqueeze(-2)).sum(-1) * scale
        G = G + q[i].unsqueeze(-1) * do.unsqueeze(-2)
        dk[i] = (G * v[i].unsqueeze(-2)).sum(-1)
        dv[i] = (G * k[i].unsqueeze(-1)).sum(-2)
        da[i] = a[i] * (G * states[i]).sum((-1, -2))
        G = a[i][..., None, None] * G
    dk, dv = (x.reshape(T, B, H // share, share, -1).sum(3) for x in (dk, dv))
    dg = da if c["decay"] == "step" else da.sum((0, 1)).reshape(1, H)
    return {"out": out, "final": S, "grads": {"q": dq, "k": dk, "v": dv, "log_decay": dg, "state": G}}


def _exact_gated(c, t):
    d = {n: None if a is None else a.double() for n, a in t.items()}
    g, u = (torch.matmul(d["x"], d[w]) + (0.0 if d[b] is None else d[b]) for w, b in (("w_gate", "b_gate"), ("w_up", "b_up")))
    act = {"relu": torch.relu, "gelu": F.gelu, "silu": F.silu, "sigmoid": torch.sigmoid}[c["act"]]
    if c["kind"] == "gated_act":
        return {"out": act(g) * u}
    g = g.requires_grad_()
    a = act(g)
    (slope,) = torch.autograd.grad(a.sum(), g)
    du, dg = d["dout"] * a.detach(), d["dout"] * u * slope
    grads = {"x": torch.matmul(dg, d["w_gate"].T) + torch.matmul(du, d["w_up"].T),
             "w_gate": torch.matmul(d["x"].T, dg), "w_up": torch.matmul(d["x"].T, du)}
    if d["b_gate"] is not None:
        grads.update(b_gate=dg.sum(0, keepdim=True), b_up=du.sum(0, keepdim=True))
    return {"out": a.detach() * u, "grads": grads}


def _exact_adamw(c, s):
    f = {n: a.double() if a.is_floating_point() else a for n, a in s["flat"].items()}
    if c["bits"] == 8:
        cm, cv = (f[n].double().reshape(-1, BLOCK) for n in ("m_codes", "v_codes"))
        f["m"] = (torch.sign(cm) * (cm / 127.0) ** 2 * f["m_scale"].reshape(-1, 1)).reshape(-1)
        f["v"] = ((cv / 255.0) ** 4 * f["v_scale"].reshape(-1, 1)).reshape(-1)
    t = STEPS_DONE + 1
    m, v = BETA1 * f["m"] + (1 - BETA1) * f["g"], BETA2 * f["v"] + (1 - BETA2) * f["g"] ** 2
    p = f["p"] - LR * (DECAY * f["p"] + (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS))
    none = [None] * len(s["shapes"])  # which of two codes a moment rounds to has no value in 64 bits
    return {"p": _split(p, s), "m": _split(m, s) if c["bits"] == 32 else none, "v": _split(v, s) if c["bits"] == 32 else none}


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "adamw":
        return _exact_adamw(case, _adamw_inputs(case, seed))
    if kind in ("gated", "gated_act"):
        return _exact_gated(case, _gated_inputs(case, seed))
    return _exact_memory(case, _memory_inputs(case, seed))


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "adamw":
        n = sum(_count(s) for s in _shapes(case))
        # parameter, gradient and both moments; in 8 bits two codes, the scales, and the values they stand for
        return {"bytes": n * (28 if case["bits"] == 32 else 12 + 4 + 4 * 4 / BLOCK + 8), "flops": 14 * n}
    if kind in ("gated", "gated_act"):
        m, i, h = case["rows"], case["in"], case["hidden"]
        weights = 2 * i * h + (2 * h if case["bias"] else 0)
        if kind == "gated_act":
            return {"bytes": 4 * (m * i + weights + m * h), "flops": 4 * m * i * h}
        return {"bytes": 4 * (2 * m * i + 2 * weights + 2 * m * h), "flops": 12 * m * i * h}
    H, G, K, V = case["heads"], case["kv_heads"], case["key"], case["value"]
    T, B = (1, case["lanes"]) if kind == "token" else (case["steps"], case["batch"])
    decays = H if case["decay"] == "head" else T * B * H
    rows, states = H * K + G * K + G * V, 2 * B * H * K * V
    reads = T * B * rows + decays + (T * B if case["done"] else 0)
    if kind != "memory":
        return {"bytes": 4 * (reads + T * B * H * V + states), "flops": 4 * T * B * H * K * V}
    grads = T * B * (rows + 2 * H * V) + decays + states // 2 * (2 if case["final_grad"] else 1)
    return {"bytes": 4 * (reads + states + grads), "flops": 12 * T * B * H * K * V}
