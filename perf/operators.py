"""The measured cases of the training and 8-bit scoring operators (include/jvgpu.h, "training and 8-bit scoring").

Two families, both products of a batch of query vectors with the rows of an index:

* ``loss`` / ``step`` / ``adapter``: softmax cross entropy of queries over all rows of an index (the loss an embedding model or a query
  adapter is tuned with against a corpus), alone, with both gradients, and with the queries' gradient alone (a frozen corpus);
* ``encode`` / ``score``: rows of 8-bit floats (e4m3) with one power-of-two scale for each block of 128 components, and the matrix product
  of a batch of queries with such rows.

With ``own`` false ``run`` computes an operator from elementary torch operations in 32 bits; with ``own`` true it calls the framework.
"""
import math

import torch

own = False

BLOCK = 128     # components that share one scale
TOP = 448.0     # the largest e4m3 value


def _ops():
    """The framework's torch view of its device operators."""
    import importlib

    import __graft_entry__ as graft
    graft.load_package()
    return importlib.import_module("opensearch_jvector_amd.ops")


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a unit test's index (10 000 x 128): one short call, launches count
        {"name": "loss-16x10000x128-f32", "kind": "loss", "nq": 16, "n": 10000, "d": 128, "dtype": "f32", "pad": 0, "scale": 20.0},
        # evaluating a batch of 256 queries against a whole index of 1M x 768
        {"name": "loss-256x1M-768-bf16", "kind": "loss", "nq": 256, "n": 1000000, "d": 768, "dtype": "bf16", "pad": 0, "scale": 20.0},
        # a small fp32 training step: in-batch size of a laptop-scale run
        {"name": "step-32x1000x64-f32", "kind": "step", "nq": 32, "n": 1000, "d": 64, "dtype": "f32", "pad": 0, "scale": 10.0},
        # an ordinary step: 1 024 queries against the sampled part of a corpus
        {"name": "step-1024x65536x768-bf16", "kind": "step", "nq": 1024, "n": 65536, "d": 768, "dtype": "bf16", "pad": 0, "scale": 20.0},
        # odd everything, fp32, rows that lie in a wider table
        {"name": "step-777x30011x381-f32", "kind": "step", "nq": 777, "n": 30011, "d": 381, "dtype": "f32", "pad": 3, "scale": 20.0},
        # the largest step
        {"name": "step-4096x131072x1024-bf16", "kind": "step", "nq": 4096, "n": 131072, "d": 1024, "dtype": "bf16", "pad": 0, "scale": 20.0},
        # tuning a query adapter against a frozen corpus of 1 536-d rows: the queries' gradient alone
        {"name": "adapter-512x200000x1536", "kind": "adapter", "nq": 512, "n": 200000, "d": 1536, "dtype": "bf16", "pad": 0, "scale": 20.0},
        # one query at a time: encode it, score 100 000 rows
        {"name": "score-1x100000x768", "kind": "score", "nq": 1, "n": 100000, "d": 768, "dtype": "f32", "out": "f32", "pad": 0},
        # 256 concurrent queries over half a million rows, every score kept
        {"name": "score-256x500000x768", "kind": "score", "nq": 256, "n": 500000, "d": 768, "dtype": "f32", "out": "f32", "pad": 0},
        # all-pairs scoring of 1 536-d vectors (a nearest-neighbour graph's exact lists): compute counts
        {"name": "score-4096x65536x1536-bf16", "kind": "score", "nq": 4096, "n": 65536, "d": 1536, "dtype": "bf16", "out": "bf16", "pad": 0},
        # a batch of queries to 8 bits and back
        {"name": "encode-256x768-f32", "kind": "encode", "n": 256, "d": 768, "dtype": "f32", "pad": 0},
        # a whole index to 8 bits and back, a row length no block divides
        {"name": "encode-1000003x1000-f32", "kind": "encode", "n": 1000003, "d": 1000, "dtype": "f32", "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["loss", "step", "adapter", "score", "encode"])
    dtype = rng.choice(["f32", "bf16"])
    pad = rng.choice([0, 0, 8, rng.randint(1, 40)])
    d = rng.choice([_log(rng, 16, 1536), 8 * _log(rng, 4, 192)])
    if kind == "encode":
        return {"kind": kind, "n": _log(rng, 16, 500000), "d": d, "dtype": dtype, "pad": pad}
    while True:
        nq, n = _log(rng, 1, 4096), _log(rng, 16, 1000000)
        if kind == "score" and n <= 500000 and nq * n <= 4096 * 65536:
            return {"kind": kind, "nq": nq, "n": n, "d": d, "dtype": dtype, "out": rng.choice(["f32", "bf16"]), "pad": pad}
        if kind != "score" and nq * n <= 4096 * 131072 // (8 if dtype == "f32" else 2):
            return {"kind": kind, "nq": nq, "n": n, "d": d, "dtype": dtype, "pad": pad, "scale": rng.choice([1.0, 10.0, 20.0, 30.0])}


def work(case):
    n, d = case["n"], case["d"]
    size = 4 if case["dtype"] == "f32" else 2
    blocks = -(-d // BLOCK)
    if case["kind"] == "encode":
        return {"bytes": 2.0 * n * (size * d + d + blocks), "flops": 4.0 * n * d}
    nq = case["nq"]
    if case["kind"] == "score":
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": nq * d * size + n * (d + blocks) + float(nq) * n * out, "flops": 2.0 * nq * n * d}
    products = {"loss": 1, "adapter": 2, "step": 3}[case["kind"]]   # the logits, and one more for each gradient
    moved = size * d * (nq + n) + 8.0 * nq
    if case["kind"] != "loss":
        moved += size * d * nq + 4 * nq
    if case["kind"] == "step":
        moved += size * d * n
    return {"bytes": moved, "flops": 2.0 * products * nq * n * d}


# ----------------------------------------------------------------------------------------------------------------- inputs
def _rows(g, n, d, pad, dtype):
    """[n][d] unit rows that lie `pad` components apart in a wider table."""
    wide = torch.randn((n, d + pad), generator=g, device="cuda")
    rows = wide[:, :d]
    rows /= rows.square().sum(1, keepdim=True).sqrt()
    return (wide.bfloat16() if dtype == "bf16" else wide)[:, :d]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, d, pad = case["n"], case["d"], case["pad"]
    if case["kind"] == "encode":
        rows = _rows(g, n, d, pad, case["dtype"])
        rows *= torch.exp2(torch.randint(-6, 7, (n, 1), generator=g, device="cuda")).to(rows.dtype)   # norms differ from row to row
        return {"case": case, "vectors": rows}
    nq = case["nq"]
    if case["kind"] == "score":
        codes, scales = _encode(_rows(g, n, d, 0, "f32"))
        return {"case": case, "queries": _rows(g, nq, d, pad, case["dtype"]), "codes": codes, "scales": scales}
    vectors = _rows(g, n, d, pad, case["dtype"])
    targets = torch.randint(0, n, (nq,), generator=g, device="cuda")
    near = 0.7 * torch.rand((nq, 1), generator=g, device="cuda")    # pairs at every stage of being learnt
    queries = _rows(g, nq, d, pad, "f32")
    wide = torch.zeros((nq, d + pad), device="cuda")
    wide[:, :d] = near * vectors[targets].float() + (1 - near * near).sqrt() * queries
    queries = (wide.bfloat16() if case["dtype"] == "bf16" else wide)[:, :d]
    targets = targets.to(torch.int32)
    if nq >= 8:
        targets[3::8] = -1                                          # queries without a known answer take no part
    weights = (targets >= 0).float() / max(1, int((targets >= 0).sum()))   # the mean over the others
    return {"case": case, "queries": queries, "vectors": vectors, "targets": targets, "weights": weights}


# ----------------------------------------------------------------------------------------------------------- plain forms
def _encode(x):
    """codes [n][blocks * 128] (e4m3 bytes, zeros behind d), scales [n][blocks] (byte b stands for 2^(b - 127))."""
    n, d = x.shape
    blocks = -(-d // BLOCK)
    v = torch.zeros((n, blocks * BLOCK), device=x.device)
    v[:, :d] = x.float()
    v = v.view(n, blocks, BLOCK)
    top = v.abs().amax(2)
    part, power = torch.frexp(top)                       # top = part * 2^power, part in [0.5, 1); 448 = 0.875 * 2^9
    power = torch.where(top == 0, torch.zeros_like(power), torch.where(part > 0.875, power - 8, power - 9)).clamp(-127, 127)
    v = v * torch.exp2(-power.float())[:, :, None]       # a power of two: exact
    _, at = torch.frexp(v)
    at = (at - 1).clamp(min=-6)                          # a value's exponent; -6 is the smallest normal one's
    steps = torch.round(v.abs() * torch.exp2((3 - at).float()))   # whole steps of 2^(at - 3), ties to the even one
    up = steps == 16                                     # rounded up to the next power of two
    at, steps = torch.where(up, at + 1, at), torch.where(up, torch.full_like(steps, 8.0), steps).int()
    byte = torch.where(steps >= 8, (at + 7) * 8 + steps - 8, steps) + torch.where(torch.signbit(v), 128, 0)
    return byte.to(torch.uint8).view(n, blocks * BLOCK), (power + 127).to(torch.uint8)


def _decode(codes, scales, d):
    low = codes.int()
    exponent, part = (low >> 3) & 15, (low & 7).float()
    value = torch.where(exponent == 0, part * 2.0 ** -9, (1 + part / 8) * torch.exp2((exponent - 7).float()))
    value = torch.where(low >= 128, -value, value)
    value = value.view(codes.shape[0], -1, BLOCK) * torch.exp2(scales.float() - 127)[:, :, None]
    return value.view(codes.shape[0], -1)[:, :d]


def _plain(state):
    case = state["case"]
    if case["kind"] == "encode":
        codes, scales = _encode(state["vectors"])
        return {"vectors": _decode(codes, scales, case["d"]).to(state["vectors"].dtype)}
    if case["kind"] == "score":
        queries = _decode(*_encode(state["queries"]), case["d"])
        scores = queries @ _decode(state["codes"], state["scales"], case["d"]).t()
        return {"scores": scores.bfloat16() if case["out"] == "bf16" else scores}
    q, v, t = state["queries"].float(), state["vectors"].float(), state["targets"].long()
    logits = (q @ v.t()) * case["scale"]
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    known = t >= 0
    at = t.clamp(min=0)[:, None]
    loss = (torch.log(total) - (logits.gather(1, at) - top))[:, 0]
    out = {"loss": torch.where(known, loss, torch.zeros_like(loss)), "lse": (torch.log(total) + top)[:, 0]}
    if case["kind"] == "loss":
        return out
    del logits
    p = p / total
    p.scatter_add_(1, at, torch.full_like(total, -1.0))
    p = p * torch.where(known, state["weights"] * case["scale"], torch.zeros_like(loss))[:, None]
    out["grad_queries"] = (p @ v).to(state["queries"].dtype)
    if case["kind"] == "step":
        out["grad_vectors"] = (p.t() @ q).to(state["vectors"].dtype)
    return out


# ------------------------------------------------------------------------------------------------------- the framework's
def _framework(state):
    ops, case = _ops(), state["case"]
    if case["kind"] == "encode":
        codes, scales = ops.encode_blocks(state["vectors"])
        return {"vectors": ops.decode_blocks(codes, scales, case["d"], state["vectors"].dtype)}
    if case["kind"] == "score":
        codes, scales = ops.encode_blocks(state["queries"])
        out = torch.bfloat16 if case["out"] == "bf16" else torch.float32
        return {"scores": ops.score_blocks(codes, scales, state["codes"], state["scales"], case["d"], out)}
    q, v, t = state["queries"], state["vectors"], state["targets"]
    loss, lse = ops.softmax_loss(q, v, t, case["scale"])
    out = {"loss": loss, "lse": lse}
    if case["kind"] != "loss":
        grads = ops.softmax_loss_grad(q, v, t, case["scale"], lse, state["weights"], queries_grad=True, vectors_grad=case["kind"] == "step", loss=loss)
        out["grad_queries"] = grads[0]
        if case["kind"] == "step":
            out["grad_vectors"] = grads[1]
    return out


def run(state):
    return _framework(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------------------------- 64 bits
def _two_to(power):
    """2^power in 64 bits, exactly (a device's pow() may be off by its last bit, which decides ties): the exponent put in place."""
    return ((power.long() + 1023) << 52).view(torch.float64)


def _nearest(x, d):
    """The values that rows of x are held as, by looking each up among all that a block can hold."""
    magnitudes = torch.tensor([m / 8.0 * 2.0 ** -6 for m in range(8)] +
                              [(1 + m / 8.0) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)],
                              dtype=torch.float64, device=x.device)
    n = x.shape[0]
    held = torch.empty((n, d), dtype=torch.float64, device=x.device)
    for lo in range(0, d, BLOCK):
        for row in range(0, n, 100000):
            part = x[row:row + 100000, lo:lo + BLOCK].double()
            top = part.abs().amax(1, keepdim=True)
            power = torch.ceil(torch.log2(torch.where(top == 0, torch.full_like(top, TOP), top) / TOP))
            power += (top > TOP * _two_to(power)).double() - (top <= TOP * _two_to(power - 1)).double() * (top > 0)
            unit = _two_to(power.clamp(min=-127))
            value = part.abs() / unit
            above = torch.searchsorted(magnitudes, value).clamp(max=len(magnitudes) - 1)
            below = (above - 1).clamp(min=0)
            gap = (magnitudes[above] - value) - (value - magnitudes[below])
            pick = torch.where((gap > 0) | ((gap == 0) & (below % 2 == 0)), below, above)
            held[row:row + 100000, lo:lo + BLOCK] = torch.sign(part) * magnitudes[pick] * unit
    return held


def exact(case, seed):
    state = prepare(case, seed)
    d = case["d"]
    if case["kind"] == "encode":
        return {"vectors": _nearest(state["vectors"], d)}
    if case["kind"] == "score":
        byte = torch.arange(128, device="cuda", dtype=torch.float64)
        e, m = torch.div(byte, 8, rounding_mode="floor"), byte % 8
        half = torch.where(e > 0, (8 + m) * _two_to(e - 10), m * 2.0 ** -9)
        table = torch.cat([half, -half])
        held = table[state["codes"].long()] * _two_to(state["scales"].long() - 127).repeat_interleave(BLOCK, 1)
        return {"scores": _nearest(state["queries"], d) @ held[:, :d].t()}
    q, v, t = state["queries"].double(), state["vectors"].double(), state["targets"].long()
    nq, step = q.shape[0], max(1, (1 << 28) // case["n"])
    loss, lses = (torch.zeros(nq, device="cuda", dtype=torch.float64) for _ in range(2))
    dq, dv = torch.zeros_like(q), torch.zeros_like(v)
    for a in range(0, nq, step):
        z = case["scale"] * (q[a:a + step] @ v.t())
        lse = torch.logsumexp(z, 1)
        known = (t[a:a + step] >= 0).double()
        rows = torch.arange(z.shape[0], device="cuda")
        at = t[a:a + step].clamp(min=0)
        lses[a:a + step] = lse
        loss[a:a + step] = known * (lse - z[rows, at])
        if case["kind"] == "loss":
            continue
        g = torch.exp(z - lse[:, None])
        g[rows, at] -= 1
        g *= (known * state["weights"][a:a + step].double() * case["scale"])[:, None]
        dq[a:a + step] = g @ v
        if case["kind"] == "step":
            dv += g.t() @ q[a:a + step]
    out = {"loss": loss, "lse": lses}
    if case["kind"] != "loss":
        out["grad_queries"] = dq
    if case["kind"] == "step":
        out["grad_vectors"] = dv
    return out
