"""Measured cases of the operators on activation rows held in 8 bits.

A row of d values is held as int8 codes with one power-of-two step per block of 32 values: ceil(d / 32) * 32 bytes of codes
(zeros behind the d-th), one byte S per block (the exponent field of the step as a float, value = code * 2^(S - 127); 0 for
a block of zeros, 255 for a block that held an infinity or a NaN), zeros up to a multiple of 16 bytes.

Four operators:
  checkpoint  rows of floats -> the 8-bit record -> the values a backward pass reads from it
  batch       rows of a buffer held in 8 bits, picked by index, scaled and cast: a shuffled training batch
  wgrad       left^T @ right over the token axis with `right` held in 8 bits: a dense weight gradient
  rows        gradient rows of a dictionary: each feature's sum of coefficient * (8-bit row of its token)

`run` gives the plain form in elementary torch operations, or, with `own`, the framework's calls.
"""

import math

import torch

own = False

BLOCK = 32
F32, BF16 = "float32", "bfloat16"


def _dtype(name):
    return torch.bfloat16 if name == BF16 else torch.float32


def _pitch(d):
    nb = -(-d // BLOCK)
    return -(-(nb * BLOCK + nb) // 16) * 16


def listed():
    return [
        # one short prompt's residual stream, kept for the backward pass: latency is what counts
        {"name": "checkpoint prompt", "op": "checkpoint", "n": 128, "d": 768, "gap": 0, "dtype": BF16},
        # the batch of the small fp32 configuration (d_model 768, 4096 tokens)
        {"name": "checkpoint fp32", "op": "checkpoint", "n": 4096, "d": 768, "gap": 0, "dtype": F32},
        # odd width, odd count, rows that are a slice of a wider tensor (one hook point of several side by side)
        {"name": "checkpoint ragged", "op": "checkpoint", "n": 5003, "d": 2049, "gap": 37, "dtype": BF16},
        # the wide configuration's rows (d_model 4096), four batches at once
        {"name": "checkpoint wide", "op": "checkpoint", "n": 16384, "d": 4096, "gap": 0, "dtype": BF16},
        # a few rows of a small buffer: the smallest batches, used in tests and on short streams
        {"name": "batch small", "op": "batch", "n": 64, "d": 768, "held": 16384, "scale": 1.0, "dtype": F32},
        # the headline batch (4096 tokens of d_model 4096) out of a shuffle buffer of 2^18 tokens
        {"name": "batch headline", "op": "batch", "n": 4096, "d": 4096, "held": 262144, "scale": 1.0, "dtype": BF16},
        # a large batch of the d_model 2048 configuration, normalised on the way out, in fp32
        {"name": "batch scaled", "op": "batch", "n": 32768, "d": 2048, "held": 131072, "scale": 0.37, "dtype": F32},
        # odd sizes: a dictionary and a batch that no tile divides
        {"name": "wgrad ragged", "op": "wgrad", "t": 1000, "m": 1003, "d": 521, "dtype": BF16},
        # the sparse attention configuration: 16 x 1024 tokens, 8192 value heads, d_model 768
        {"name": "wgrad attention heads", "op": "wgrad", "t": 16384, "m": 8192, "d": 768, "dtype": BF16},
        # a dense (threshold) dictionary of d_model 2048, 32768 features, 8192 tokens
        {"name": "wgrad dense dictionary", "op": "wgrad", "t": 8192, "m": 32768, "d": 2048, "dtype": BF16},
        # the small configuration: 4096 tokens, 32 of 6144 features each
        {"name": "rows small", "op": "rows", "t": 4096, "k": 32, "f": 6144, "d": 768},
        # the middle configuration: 8192 tokens, 64 of 32768 features each
        {"name": "rows middle", "op": "rows", "t": 8192, "k": 64, "f": 32768, "d": 2048},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["checkpoint", "batch", "wgrad", "rows"])
    dtype = rng.choice([F32, BF16])
    if op == "checkpoint":
        d = _spread(rng, 32, 4096)
        return {"op": op, "n": _spread(rng, 1, (1 << 25) // d), "d": d, "gap": rng.choice([0, 0, rng.randrange(1, 64)]), "dtype": dtype}
    if op == "batch":
        d = _spread(rng, 32, 4096)
        return {"op": op, "n": _spread(rng, 1, (1 << 25) // d), "d": d, "held": _spread(rng, 1024, (1 << 28) // d),
                "scale": rng.choice([1.0, rng.uniform(0.05, 20.0)]), "dtype": dtype}
    if op == "wgrad":
        d = _spread(rng, 32, 2048)
        m = _spread(rng, 32, 8192)
        return {"op": op, "t": _spread(rng, 1, 8192), "m": m, "d": d, "dtype": rng.choice([BF16, BF16, F32]) if m <= 2048 else BF16}
    d = _spread(rng, 32, 2048)
    f = _spread(rng, 256, 32768)
    return {"op": op, "t": _spread(rng, 1, 8192), "k": _spread(rng, 1, 64), "f": f, "d": d}


# ---- inputs ----------------------------------------------------------------------------------------


def _activations(n, d, gen):
    """[n, d] fp32 rows like a residual stream's: a token-wise spread of norms and a few outlier dimensions."""
    x = torch.randn(n, d, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(n, 1, generator=gen, device="cuda"))
    x[:, torch.randint(0, d, (max(1, d // 1024),), generator=gen, device="cuda")] *= 40.0
    return x


def _held(x, d):
    """The 8-bit rows of x [n, d] (fp32): uint8 [n, pitch]."""
    n, nb = x.shape[0], -(-d // BLOCK)
    full = torch.zeros(n, nb * BLOCK, device=x.device)
    full[:, :d] = x
    blocks = full.view(n, nb, BLOCK)
    step_field = _step_field(blocks.abs().amax(2))
    codes = torch.round(blocks * _power(127 - step_field)[:, :, None]).clamp(-127, 127).to(torch.int8)
    rows = torch.zeros(n, _pitch(d), dtype=torch.uint8, device=x.device)
    rows[:, : nb * BLOCK] = codes.view(n, nb * BLOCK).view(torch.uint8)
    rows[:, nb * BLOCK : nb * BLOCK + nb] = step_field.to(torch.uint8)
    return rows


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "checkpoint":
        wide = _activations(case["n"], case["d"] + case["gap"], gen).to(_dtype(case["dtype"]))
        return {"op": op, "x": wide[:, : case["d"]]}
    d = case["d"]
    if op == "batch":
        # a buffer of as many distinct rows as is quick to make, repeated up to its size in another order
        held, distinct = case["held"], min(case["held"], max(1, (1 << 25) // d))
        rows = _held(_activations(distinct, d, gen), d)
        if held > distinct:
            rows = rows[torch.randint(0, distinct, (held,), generator=gen, device="cuda")]
        idx = torch.randint(0, held, (case["n"],), generator=gen, device="cuda")
        return {"op": op, "rows": rows, "d": d, "idx": idx, "scale": case["scale"], "dtype": _dtype(case["dtype"])}
    rows = _held(_activations(case["t"], d, gen), d)
    if op == "wgrad":
        # gradients at the pre-activations: small, with a token-wise spread
        left = torch.randn(case["t"], case["m"], generator=gen, device="cuda") * 1e-3
        left *= torch.exp(torch.randn(case["t"], 1, generator=gen, device="cuda"))
        return {"op": op, "left": left.to(_dtype(case["dtype"])), "rows": rows, "d": d}
    # k distinct features of every token, a few of them far more frequent than most, in ascending order
    t, f = case["t"], case["f"]
    k = min(case["k"], f)
    often = -1.2 * torch.log(torch.arange(1, f + 1, device="cuda", dtype=torch.float32))
    order = torch.randperm(f, generator=gen, device="cuda")
    noise = torch.rand(t, f, generator=gen, device="cuda").clamp_(1e-20, 1 - 1e-7)
    idx = torch.topk(often[order] - torch.log(-torch.log(noise)), k, dim=1).indices.sort(1).values
    coef = torch.randn(t * k, generator=gen, device="cuda") * 1e-3
    flat = idx.reshape(-1)
    # the index of the code by feature (slots in ascending order), which a step builds once for both weight matrices
    slot = torch.sort(flat, stable=True).indices.to(torch.int32)
    ptr = torch.zeros(f + 1, dtype=torch.int32, device="cuda")
    ptr[1:] = torch.cumsum(torch.bincount(flat, minlength=f), 0).to(torch.int32)
    tok = (torch.arange(t * k, device="cuda") // k).to(torch.int32)
    return {"op": op, "rows": rows, "d": d, "f": f, "feature": flat, "coef": coef, "ptr": ptr, "slot": slot, "tok": tok}


# ---- the plain form ----------------------------------------------------------------------------------


def _step_field(amax):
    """S of blocks with these largest magnitudes (fp32), as int32."""
    bits = amax.view(torch.int32)
    field, mantissa = bits >> 23, bits & 0x7FFFFF
    bump = (field >= 7) & (field < 254) & (mantissa >= 0x7F0000)
    s = torch.clamp(field - 6, min=1) + bump.to(torch.int32)
    s = torch.where(bits == 0, torch.zeros_like(s), s)
    return torch.where(field == 255, torch.full_like(s, 255), s)


def _power(field):
    """2^field' for a scaling exponent: 2^(field) through the float's own bits (0 and below give 0)."""
    return (torch.clamp(field + 127, 0, 254) << 23).view(torch.float32)


def _values(rows, d):
    """fp32 [n, d] of 8-bit rows."""
    n, nb = rows.shape[0], -(-d // BLOCK)
    codes = rows[:, : nb * BLOCK].view(torch.int8).float().view(n, nb, BLOCK)
    step = (rows[:, nb * BLOCK : nb * BLOCK + nb].to(torch.int32) << 23).view(torch.float32)
    return (codes * step[:, :, None]).view(n, nb * BLOCK)[:, :d]


def run(state):
    op = state["op"]
    if own:
        return _own(state)
    if op == "checkpoint":
        x = state["x"]
        return _values(_held(x.float(), x.shape[1]), x.shape[1]).to(x.dtype)
    if op == "batch":
        return (_values(state["rows"].index_select(0, state["idx"]), state["d"]) * state["scale"]).to(state["dtype"])
    if op == "wgrad":
        return state["left"].float().t() @ _values(state["rows"], state["d"])
    contribution = state["coef"][:, None] * _values(state["rows"], state["d"])[state["tok"].long()]
    out = torch.zeros(state["f"], state["d"], device=contribution.device)
    return out.index_add_(0, state["feature"], contribution)


def _own(state):
    from __graft_entry__ import load_package

    ops = load_package().ops
    op = state["op"]
    if op == "checkpoint":
        x = state["x"]
        return ops.restore_rows(ops.quantize_rows(x), x.dtype)
    rows = ops.Rows8(state["rows"], state["d"])
    if op == "batch":
        return ops.gather_rows(rows, state["idx"], state["dtype"], state["scale"])
    if op == "wgrad":
        return ops.gemm_over_tokens(state["left"], rows, torch.float32)
    fi = ops.FeatureIndex(state["ptr"], state["slot"], state["tok"])
    return ops.sparse_grad_rows(fi, state["coef"], rows, state["f"])[0]


# ---- what a pass cannot do without, and its exact result -------------------------------------------------


def work(case):
    d = case["d"]
    held = -(-d // BLOCK) * (BLOCK + 1)
    size = 2 if case.get("dtype") == BF16 else 4
    if case["op"] == "checkpoint":  # read, recorded, the record read again, values written
        return {"bytes": case["n"] * (2 * size * d + 2 * held), "flops": 6 * case["n"] * d}
    if case["op"] == "batch":
        return {"bytes": case["n"] * (held + 8 + size * d), "flops": 2 * case["n"] * d}
    if case["op"] == "wgrad":
        t, m = case["t"], case["m"]
        return {"bytes": t * m * size + t * held + 4 * m * d, "flops": 2 * t * m * d}
    slots = case["t"] * min(case["k"], case["f"])
    return {"bytes": case["t"] * held + 12 * slots + 4 * case["f"] * (d + 1), "flops": 2 * slots * d}


def _exact_values(rows, d):
    """fp64 [n, d]: code times two to the power S - 127, column by column of the record."""
    column = torch.arange(d, device=rows.device)
    code = rows[:, :d].to(torch.float64)
    code = torch.where(code > 127, code - 256, code)
    field = rows[:, -(-d // BLOCK) * BLOCK :][:, column // BLOCK].to(torch.float64)
    return torch.where(field == 0, torch.zeros_like(code), code * torch.exp2(field - 127))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "checkpoint":
        x = state["x"].double()
        n, d = x.shape
        pad = -d % BLOCK
        blocks = torch.cat([x, torch.zeros(n, pad, dtype=torch.float64, device=x.device)], 1).reshape(n, -1, BLOCK)
        top = blocks.abs().max(2, keepdim=True).values
        # the smallest power of two that brings the largest magnitude to 127 after rounding (ties to even)
        step = torch.exp2(torch.floor(torch.log2(top.clamp_min(2.0**-120))) - 6)
        step = torch.where(torch.round(top / step) > 127, 2 * step, step)
        return (torch.round(blocks / step) * step).reshape(n, -1)[:, :d]
    values = _exact_values(state["rows"], state["d"])
    if case["op"] == "batch":
        return values[state["idx"]] * state["scale"]
    if case["op"] == "wgrad":
        return state["left"].double().t() @ values
    code = torch.zeros(case["t"], case["f"], dtype=torch.float64, device="cuda")
    code[state["tok"].long(), state["feature"]] = state["coef"].double()
    return code.t() @ values
