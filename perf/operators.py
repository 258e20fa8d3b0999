"""Products of BF16 activations with weights held in packed E2M1 (4-bit) and block scales, as a serving loop calls them.

    dense    D[M, N] = A[M, K] @ W[N, K]^T                      one weight matrix (a projection of a decode or prefill step)
    ragged   D[r, :] = A[r, :] @ W[g(r), N, K]^T                rows sorted by expert, group sizes as they fall, no padding rows

A is bfloat16.  W[n, k] = e2m1(code[n, k]) * 2^(e[n, k // gran] - 127): two codes per byte, the even k in the low nibble, one
power-of-two scale (UE8M0) per `gran` elements of k, four scales to an int32 word, words MN-major ([N, ceil(K / (4 gran))] with
strides (1, align(N, 4)), experts one after another): what the FP8 x FP4 GEMMs of the package take for the same weights.
`group_ends[g]` (int32, on the device) is the row where group g ends; group g starts where group g - 1 ends.  Rows at or behind
the last end belong to no group and keep what D holds.
"""
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def listed():
    """Shapes are those of the package's benchmark: the six (N, K) of its dense GEMMs, the 32- and 16-expert layers of its grouped ones."""
    return [
        # one token of a single sequence through the narrowest and through the largest weight matrix: latency, then bandwidth
        {"name": "dense m1 n2112 k7168", "op": "dense", "m": 1, "n": 2112, "k": 7168, "gran": 32, "out": "bf16"},
        {"name": "dense m1 n7168 k16384", "op": "dense", "m": 1, "n": 7168, "k": 16384, "gran": 32, "out": "bf16"},
        # a few sequences decoding together (an odd number of rows), weights with one scale per 128 elements
        {"name": "dense m7 n24576 k1536", "op": "dense", "m": 7, "n": 24576, "k": 1536, "gran": 128, "out": "bf16"},
        # a decode batch whose output stays in FP32 (logits, or a router's input)
        {"name": "dense m16 n4096 k7168 fp32", "op": "dense", "m": 16, "n": 4096, "k": 7168, "gran": 32, "out": "fp32"},
        # larger decode batches and a short prompt, odd row counts
        {"name": "dense m61 n7168 k2048", "op": "dense", "m": 61, "n": 7168, "k": 2048, "gran": 32, "out": "bf16"},
        {"name": "dense m500 n32768 k512", "op": "dense", "m": 500, "n": 32768, "k": 512, "gran": 128, "out": "bf16"},
        # a prefill chunk
        {"name": "dense m4096 n7168 k2048", "op": "dense", "m": 4096, "n": 7168, "k": 2048, "gran": 32, "out": "bf16"},
        # a small expert layer: most groups of a few rows, one empty
        {"name": "ragged g4 r37 n2112 k1536", "op": "ragged", "groups": 4, "active": 3, "rows": 37, "spare": 3, "n": 2112, "k": 1536, "gran": 128},
        # one token routed to 8 of 32 experts
        {"name": "ragged g32 r8 n4096 k7168", "op": "ragged", "groups": 32, "active": 8, "rows": 8, "spare": 0, "n": 4096, "k": 7168, "gran": 32},
        # a decode batch, some experts crowded and some empty
        {"name": "ragged g32 r131 n7168 k2048", "op": "ragged", "groups": 32, "active": 24, "rows": 131, "spare": 5, "n": 7168, "k": 2048, "gran": 32},
        # a large decode batch: about 61 rows to each of 16 experts
        {"name": "ragged g16 r972 n4096 k7168", "op": "ragged", "groups": 16, "active": 16, "rows": 972, "spare": 0, "n": 4096, "k": 7168, "gran": 32},
        # a prefill chunk through an expert layer
        {"name": "ragged g32 r8191 n4096 k7168", "op": "ragged", "groups": 32, "active": 31, "rows": 8191, "spare": 1, "n": 4096, "k": 7168, "gran": 32},
    ]


def draw(rng):
    """Rows from one to thousands, N in steps of 8, K in steps of 128, both scale granularities, groups empty or crowded; no case
    reads more weights or multiplies more than the largest listed one."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    gran = rng.choice((32, 128))
    if rng.random() < 0.5:
        while True:
            m, n, k = spread(1, 4096), 8 * spread(4, 4096), 128 * spread(1, 128)
            if n * k <= 7168 * 16384 and m * n * k <= 4096 * 7168 * 2048:
                return {"op": "dense", "m": m, "n": n, "k": k, "gran": gran, "out": "fp32" if rng.random() < 0.25 else "bf16"}
    while True:
        groups = spread(2, 64)
        active, rows = rng.randint(max(1, groups // 4), groups), spread(1, 8191)
        n, k = 8 * spread(16, 896), 128 * spread(1, 56)
        if rows >= active and groups * n * k <= 32 * 4096 * 7168 and rows * n * k <= 8191 * 4096 * 7168:
            return {"op": "ragged", "groups": groups, "active": active, "rows": rows, "spare": rng.choice((0, 0, rng.randint(1, 9))), "n": n, "k": k, "gran": gran}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, k, g):
    """Rows of differing magnitude with a few large channels, as the residual stream of a trained model has them."""
    x = torch.randn((rows, k), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=g, device="cuda"))
    x *= torch.where(torch.rand((1, k), generator=g, device="cuda") < 0.005, 20.0, 1.0)
    return x.to(torch.bfloat16)


def _weights(groups, n, k, gran, g):
    """Packed codes int8 [groups, n, k / 2] and packed scales int32 [groups, n, ceil(k / (4 gran))], MN-major."""
    codes = torch.randint(0, 256, (groups, n, k // 2), generator=g, device="cuda", dtype=torch.uint8).view(torch.int8)
    pitch, words = (n + 3) // 4 * 4, -(-k // (4 * gran))
    exps = torch.randint(112, 121, (groups, words, pitch, 4), generator=g, device="cuda", dtype=torch.uint8)
    last = torch.arange(words * 4, device="cuda").view(1, words, 1, 4) < -(-k // gran)
    packed = (exps * last).contiguous().view(torch.int32).view(groups, words, pitch)
    return codes, packed.transpose(1, 2)[:, :n]


def _counts(case, g):
    """Rows per group: `active` groups get at least one each, the rest of the rows falls unevenly among them."""
    groups, active, rows = case["groups"], case["active"], case["rows"]
    chosen = torch.randperm(groups, generator=g, device="cuda")[:active]
    weight = torch.empty(active, device="cuda").exponential_(generator=g) + 0.2
    extra = torch.multinomial(weight, max(1, rows - active), replacement=True, generator=g)[: rows - active]
    counts = torch.zeros(groups, dtype=torch.int64, device="cuda")
    counts[chosen] = 1 + torch.bincount(extra, minlength=active)
    return counts


def prepare(case, seed):
    g = _generator(seed)
    n, k, gran = case["n"], case["k"], case["gran"]
    if case["op"] == "dense":
        w, sf = _weights(1, n, k, gran, g)
        return {"case": case, "a": _activations(case["m"], k, g), "w": w[0], "sf": sf[0],
                "d": torch.zeros((case["m"], n), dtype=torch.float32 if case["out"] == "fp32" else torch.bfloat16, device="cuda")}
    w, sf = _weights(case["groups"], n, k, gran, g)
    counts = _counts(case, g)
    rows = case["rows"] + case["spare"]
    return {"case": case, "a": _activations(rows, k, g), "w": w, "sf": sf, "group_ends": counts.cumsum(0).to(torch.int32),
            "most": int(counts.max()), "d": torch.zeros((rows, n), dtype=torch.bfloat16, device="cuda")}


def _dequantised(w, sf, k, gran):
    """W in FP32: [..., n, k]."""
    w = w.view(torch.uint8)
    codes = torch.stack((w & 15, w >> 4), -1).flatten(-2)
    values = torch.tensor(E2M1, device=w.device)[codes.int()]
    shifts = torch.arange(0, 32, 8, device=w.device, dtype=torch.int32)
    exps = ((sf.unsqueeze(-1) >> shifts) & 255).flatten(-2)[..., : -(-k // gran)]
    scales = torch.exp2((exps - 127).float())
    return values * scales.repeat_interleave(gran, -1)[..., :k]


def run(state):
    case, a, w, sf, d = (state[x] for x in ("case", "a", "w", "sf", "d"))
    k, gran = case["k"], case["gran"]
    if own:
        import deepgemm_amd_b200 as dg
        if case["op"] == "dense":
            dg.bf16_fp4_gemm_nt(a, (w, sf), d, recipe_b=(1, gran))
        else:
            dg.m_grouped_bf16_fp4_gemm_nt_ragged(a, (w, sf), d, state["group_ends"], recipe_b=(1, gran))
        return d
    if case["op"] == "dense":
        return (a.float() @ _dequantised(w, sf, k, gran).T).to(d.dtype)
    # Every group's rows side by side in a padded batch, one batched product, and the rows back where they came from
    ends, rows = state["group_ends"].long(), a.size(0)
    row = torch.arange(rows, device=a.device)
    group = torch.searchsorted(ends, row, right=True)
    used = (group < case["groups"]).unsqueeze(1)
    group = group.clamp(max=case["groups"] - 1)
    place = (row - (ends[group] - torch.diff(ends, prepend=ends.new_zeros(1))[group])).clamp(max=state["most"] - 1)
    padded = torch.zeros((case["groups"], state["most"], k), device=a.device)
    padded.index_put_((group, place), torch.where(used, a.float(), 0.0), accumulate=True)
    out = torch.bmm(padded, _dequantised(w, sf, k, gran).transpose(1, 2))[group, place]
    return torch.where(used, out, 0.0).to(d.dtype)


def work(case):
    n, k, gran = case["n"], case["k"], case["gran"]
    one = n * k // 2 + n * -(-k // gran)
    if case["op"] == "dense":
        m, matrices, out = case["m"], 1, 4 if case["out"] == "fp32" else 2
    else:
        m, matrices, out = case["rows"], case["active"], 2
    return {"bytes": matrices * one + m * k * 2 + m * n * out, "flops": 2 * m * n * k}


def exact(case, seed):
    """The same products in 64 bits: magnitudes from the code's exponent and mantissa bits, scales as powers of two, one group at a time."""
    state = prepare(case, seed)
    a, k, gran = state["a"].double(), case["k"], case["gran"]

    def product(x, w, sf):
        w = w.to(torch.int16) & 255
        y = torch.empty((w.size(0), k), dtype=torch.float64, device=w.device)
        for half in (0, 1):
            code = (w >> (4 * half)) & 15
            exponent, mantissa = (code >> 1) & 3, (code & 1).double()
            size = torch.where(exponent == 0, 0.5 * mantissa, (1.0 + 0.5 * mantissa) * 2.0 ** (exponent - 1).double())
            y[:, half::2] = torch.where(code >= 8, -size, size)
        for block in range(-(-k // gran)):
            e = (sf[:, block // 4].long() >> (8 * (block % 4))) & 255
            y[:, block * gran:(block + 1) * gran] *= torch.ldexp(torch.ones_like(e, dtype=torch.float64), e - 127).unsqueeze(1)
        return x @ y.T

    if case["op"] == "dense":
        return product(a, state["w"], state["sf"])
    out = torch.zeros((a.size(0), case["n"]), dtype=torch.float64, device="cuda")
    start = 0
    for group, end in enumerate(state["group_ends"].tolist()):
        if end > start:
            out[start:end] = product(a[start:end], state["w"][group], state["sf"][group])
        start = max(start, end)
    return out
