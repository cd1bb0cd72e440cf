"""Timed cases of the training operators around the PEER layer: layer norm
(forward and backward), row-scaled 8-bit activation checkpoints, and the scaled
embedding lookup with its gradient.

Every case exists twice: in plain form (elementary torch operations in 32
bits, rounded once at the end) and, with ``own`` true, as the calls a training
program makes of ``llm720_b200``.  ``exact`` gives the same outputs from the
definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_EPS = 1e-5
_E4M3_MAX = 448.0


def listed():
    return [
        # the norm in front of a layer, one decoding step of 64 sequences
        dict(name="norm_infer_64x4096_bf16", op="norm", train=False, ck=False, rows=64, dim=4096, dtype="bfloat16",
             param="float32"),
        # a small layer trained in fp32 (two sequences of 128 tokens)
        dict(name="norm_train_256x256_f32", op="norm", train=True, ck=False, rows=256, dim=256, dtype="float32",
             param="float32"),
        # the norm of a 2048-wide block, eight sequences of 2048 tokens, fp32 parameters
        dict(name="norm_train_16384x2048_bf16", op="norm", train=True, ck=False, rows=16384, dim=2048, dtype="bfloat16",
             param="float32"),
        # an odd width and a ragged batch, parameters in the activations' type
        dict(name="norm_train_5003x1537_f16", op="norm", train=True, ck=False, rows=5003, dim=1537, dtype="float16",
             param="float16"),
        # the same block norm, its input kept for the backward pass in 8 bits
        dict(name="norm_ck_16384x2048_bf16", op="norm", train=True, ck=True, rows=16384, dim=2048, dtype="bfloat16",
             param="float32"),
        # wide fp32 rows kept in 8 bits, a ragged batch
        dict(name="norm_ck_1031x4100_f32", op="norm", train=True, ck=True, rows=1031, dim=4100, dtype="float32",
             param="float32"),
        # a block's input packed in the forward pass and unpacked in the backward pass
        dict(name="pack_16384x2048_bf16", op="pack", rows=16384, dim=2048, dtype="bfloat16"),
        # the same of a small ragged fp32 tensor
        dict(name="pack_777x1001_f32", op="pack", rows=777, dim=1001, dtype="float32"),
        # token lookup of one decoding step
        dict(name="embed_infer_64_32000x4096_bf16", op="embed", train=False, tokens=64, vocab=32000, dim=4096,
             dtype="bfloat16", zipf=False, masked=0.0, padding=False),
        # a training batch of uniformly drawn token ids
        dict(name="embed_train_16384_32000x2048_bf16", op="embed", train=True, tokens=16384, vocab=32000, dim=2048,
             dtype="bfloat16", zipf=False, masked=0.0, padding=False),
        # text-like id frequencies, padded positions masked out, a small odd vocabulary in fp32
        dict(name="embed_train_30011_4001x520_f32", op="embed", train=True, tokens=30011, vocab=4001, dim=520,
             dtype="float32", zipf=True, masked=0.2, padding=True),
        # a large batch of text-like ids: some rows collect thousands of tokens
        dict(name="embed_train_131072_32000x2048_bf16", op="embed", train=True, tokens=131072, vocab=32000, dim=2048,
             dtype="bfloat16", zipf=True, masked=0.0, padding=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "pack", "embed", "embed"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    dim = _log_int(rng, 32, 8192)
    if rng.random() < 0.6:
        dim = max(32, dim // 32 * 32)                      # widths of models are mostly multiples of 32
    limit = 16384 * 2048 * (2 if dtype == "float32" else 4) // 2      # elements of the largest activations drawn
    rows = min(_log_int(rng, 1, 32768), limit // dim)
    if op == "norm":
        return dict(op="norm", train=rng.random() < 0.8, ck=rng.random() < 0.4, rows=rows, dim=dim, dtype=dtype,
                    param=rng.choice(["float32", dtype]))
    if op == "pack":
        return dict(op="pack", rows=rows, dim=dim, dtype=dtype)
    vocab = min(_log_int(rng, 2, 131072), limit // dim)
    return dict(op="embed", train=rng.random() < 0.8, tokens=rows, vocab=max(2, vocab), dim=dim, dtype=dtype,
                zipf=rng.random() < 0.5, masked=rng.choice([0.0, 0.0, 0.3]), padding=rng.random() < 0.5)


def _activations(gen, rows, dim, dtype):
    """A residual stream: rows of different size, a few channels far larger than the rest, now and then a padded
    (all-zero) row."""
    x = torch.randn(rows, dim, generator=gen, device="cuda")
    channel = torch.rand(dim, generator=gen, device="cuda")
    x *= torch.where(channel < 0.005, 24.0, 1.0)
    x += 0.3 * torch.randn(dim, generator=gen, device="cuda")
    x *= 0.5 + 2.0 * torch.rand(rows, 1, generator=gen, device="cuda")
    x *= (torch.rand(rows, 1, generator=gen, device="cuda") > 0.01)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    state = dict(case=dict(case))
    if case["op"] == "embed":
        tokens, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        u = torch.rand(tokens, generator=gen, device="cuda", dtype=torch.float64)
        if case["zipf"]:                                   # frequency ~ 1 / rank, ranks scattered over the vocabulary
            rank = (torch.exp(u * math.log(vocab)) - 1.0).long().clamp_(0, vocab - 1)
            ids = torch.randperm(vocab, generator=gen, device="cuda")[rank]
        else:
            ids = (u * vocab).long().clamp_(0, vocab - 1)
        if case["masked"] > 0:                             # positions that hold no token
            ids[torch.rand(tokens, generator=gen, device="cuda") < case["masked"]] = -1
        state["ids"] = ids
        state["padding_idx"] = 1 if case["padding"] else None
        state["scale"] = math.sqrt(dim)
        state["weight"] = (0.02 * torch.randn(vocab, dim, generator=gen, device="cuda")).to(dtype)
        if case["train"]:
            state["weight"].requires_grad_()
            state["grad"] = (0.05 * torch.randn(tokens, dim, generator=gen, device="cuda")).to(dtype)
        return state
    rows, dim = case["rows"], case["dim"]
    state["x"] = _activations(gen, rows, dim, dtype)
    if case["op"] == "norm":
        param = _DTYPES[case["param"]]
        state["weight"] = (1.0 + 0.2 * torch.randn(dim, generator=gen, device="cuda")).to(param)
        state["bias"] = (0.1 * torch.randn(dim, generator=gen, device="cuda")).to(param)
        if case["train"]:
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
            state["grad"] = (0.05 * torch.randn(rows, dim, generator=gen, device="cuda")).to(dtype)
    return state


# ---------------------------------------------------------------- the framework's calls

def _run_own(state):
    import llm720_b200 as lib
    case = state["case"]
    if case["op"] == "pack":
        payload, scale = lib.pack_rows_e4m3(state["x"])
        return lib.unpack_rows_e4m3(payload, scale, state["x"].dtype), scale
    if case["op"] == "norm":
        x, w, b = state["x"], state["weight"], state["bias"]
        if not case["train"]:
            with torch.no_grad():
                return lib.layer_norm(x, w, b, _EPS)
        y = lib.layer_norm(x, w, b, _EPS, checkpoint="e4m3" if case["ck"] else None)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), state["grad"]))
    ids, w = state["ids"], state["weight"]
    if not case["train"]:
        with torch.no_grad():
            return lib.embedding(ids, w, state["scale"], padding_idx=state["padding_idx"])
    out = lib.embedding(ids, w, state["scale"], padding_idx=state["padding_idx"])
    return (out.detach(), *torch.autograd.grad(out, (w,), state["grad"]))


# ---------------------------------------------------------------- plain forms, 32 bits

def _packed(x):
    """Row-scaled 8-bit values of fp32 x: (payload, scale); scale is the smallest power of two that brings the row
    into the format's range, 1 for a row of zeros."""
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dim=-1, keepdim=True)
    mantissa, exponent = torch.frexp(top / _E4M3_MAX)
    exponent = torch.where(mantissa > 0.5, exponent, exponent - 1).clamp_min(-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), exponent), torch.ones_like(top))
    return torch.where(torch.isfinite(x), x / scale, math.nan).to(torch.float8_e4m3fn), scale


def _unpacked(payload, scale, dtype):
    top = torch.finfo(dtype).max
    return (payload.float() * scale).clamp(-top, top)


def _run_plain(state):
    case = state["case"]
    dtype = _DTYPES[case["dtype"]]
    with torch.no_grad():
        if case["op"] == "pack":
            payload, scale = _packed(state["x"].float())
            return _unpacked(payload, scale, dtype).to(dtype), scale.squeeze(-1)
        if case["op"] == "norm":
            x, w, b = state["x"].float(), state["weight"].float(), state["bias"].float()
            mean = x.mean(dim=-1, keepdim=True)
            centred = x - mean
            rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=-1, keepdim=True) + _EPS)
            y = (centred * rstd * w + b).to(dtype)
            if not case["train"]:
                return y
            if case["ck"]:
                centred = _unpacked(*_packed(x), dtype) - mean
            dy = state["grad"].float()
            norm = centred * rstd
            g = dy * w
            dx = rstd * (g - g.mean(dim=-1, keepdim=True) - norm * (g * norm).mean(dim=-1, keepdim=True))
            return (y, dx.to(dtype), (dy * norm).sum(dim=0).to(state["weight"].dtype),
                    dy.sum(dim=0).to(state["bias"].dtype))
        ids, w = state["ids"], state["weight"]
        real = (ids >= 0) & (ids < case["vocab"])
        safe = torch.where(real, ids, 0)
        out = (torch.where(real.unsqueeze(-1), w[safe].float(), 0.0) * state["scale"]).to(dtype)
        if not case["train"]:
            return out
        if state["padding_idx"] is not None:
            real = real & (ids != state["padding_idx"])
        total = torch.zeros(case["vocab"], case["dim"], device=w.device)
        total.index_add_(0, safe, torch.where(real.unsqueeze(-1), state["grad"].float(), 0.0))
        return out, (total * state["scale"]).to(dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- 64 bits, from the definitions

def _exact_e4m3(x):
    """Values that the 8-bit form of x (64 bits, finite) stands for, and the rows' scales."""
    top = x.abs().amax(dim=-1, keepdim=True)
    power = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / _E4M3_MAX)) - 1.0     # then corrected upwards
    for _ in range(2):
        power = torch.where(top > _E4M3_MAX * torch.exp2(power), power + 1.0, power)
    scale = torch.where(top > 0, torch.exp2(power.clamp_min(-126.0)), 1.0)
    v = x / scale
    # 3 stored bits of mantissa; exponents below -6 share the spacing 2^-9; torch.round goes to even on ties
    octave = torch.frexp(v)[1].double() - 1.0
    step = torch.exp2(octave.clamp_min(-6.0) - 3.0)
    return torch.round(v / step) * step * scale, scale


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "pack":
            value, scale = _exact_e4m3(state["x"].double())
            top = torch.finfo(state["x"].dtype).max
            return value.clamp(-top, top), scale.squeeze(-1)
        if case["op"] == "norm":
            x, w, b = (state[k].detach().double() for k in ("x", "weight", "bias"))
            n = case["dim"]
            mean = x.sum(dim=1) / n
            var = ((x - mean[:, None]) ** 2).sum(dim=1) / n
            sigma = torch.sqrt(var + _EPS)
            y = (x - mean[:, None]) / sigma[:, None] * w + b
            if not case["train"]:
                return y
            if case["ck"]:
                top = torch.finfo(_DTYPES[case["dtype"]]).max
                x = _exact_e4m3(x)[0].clamp(-top, top)
            h = (x - mean[:, None]) / sigma[:, None]
            dy = state["grad"].double()
            a = torch.mv(dy, w) / n                        # mean of dy w over the row
            c = torch.mv(dy * h, w) / n                    # mean of dy w h over the row
            dx = (dy * w - a[:, None] - h * c[:, None]) / sigma[:, None]
            return y, dx, torch.einsum("rd,rd->d", dy, h), dy.sum(dim=0)
        ids, w = state["ids"], state["weight"].detach()
        inside = (ids >= 0) & (ids < case["vocab"])
        out = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device=w.device)
        out[inside] = w[ids[inside]].double() * state["scale"]
        if not case["train"]:
            return out
        if state["padding_idx"] is not None:
            inside &= ids != state["padding_idx"]
        grad = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device=w.device)
        grad.index_put_((ids[inside],), state["grad"][inside].double() * state["scale"], accumulate=True)
        return out, grad


def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    if case["op"] == "embed":
        tokens, dim, vocab = case["tokens"], case["dim"], case["vocab"]
        moved = tokens * 8 + tokens * dim * size + min(tokens, vocab) * dim * size
        ops = tokens * dim
        if case["train"]:
            moved += tokens * dim * size + vocab * dim * size
            ops += tokens * dim + vocab * dim
        return {"bytes": moved, "flops": ops}
    elements = case["rows"] * case["dim"]
    if case["op"] == "pack":
        return {"bytes": elements * (2 * size + 2) + 8 * case["rows"], "flops": 4 * elements}
    params = case["dim"] * {"float32": 4, "bfloat16": 2, "float16": 2}[case["param"]]
    if not case["train"]:
        return {"bytes": 2 * elements * size + 2 * params, "flops": 8 * elements}
    return {"bytes": 4 * elements * size + 4 * params, "flops": 20 * elements}
