"""Cases on which the operators for matrices in 4 bits are measured: quantisation, dequantisation and the two products.

Two microscaled formats of e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), values along k sharing a scale in groups:
  nvfp4  groups of 16, scale in e4m3, and a power of two for every row: the least 2^j (j >= -100) with amax(row) <= 2688 * 2^j
         (2688 = 6 * 448; 1 for a row of zeros); scale = e4m3(gmax / 6 / 2^j), code = e2m1(x / (scale * 2^j)), 0 where scale is 0
  mxfp4  groups of 32, scale 2^e with e = floor(log2(gmax)) - 2 in [-127, 127], code = e2m1(x / 2^e)
All roundings are to nearest, ties to even; codes saturate at 6.  In a matrix of 16 x 16 blocks a group is a row of a block
(nvfp4), or the row of an aligned pair of blocks, an absent one counting as zeros (mxfp4).

Operators ("op")
  dense    activations [N][K] to 4 bits and back (what the quantised layer sees of them)
  blocks   the stored blocks of a block-sparse layer to 4 bits and back
  decode   C = A x B with the layer in 4 bits and the activations in 16 bits (a few tokens: all weights are read for them)
  prefill  the same with activations that arrive in 16 bits and are quantised in the pass (many tokens)
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # One token's activations: the smallest call, latency decides.
        {"name": "dense_token", "op": "dense", "fmt": "nvfp4", "dtype": "float16", "N": 1, "K": 28672},
        # A prompt of 4096 tokens before the largest layer.
        {"name": "dense_prompt", "op": "dense", "fmt": "nvfp4", "dtype": "bfloat16", "N": 4096, "K": 28672},
        # fp32 activations at sizes that divide nothing, half a group at the end of every row.
        {"name": "dense_ragged", "op": "dense", "fmt": "mxfp4", "dtype": "float32", "N": 333, "K": 8176},
        # The weights of the benchmark's block-sparse layer, when they are brought into 4 bits.
        {"name": "blocks_layer", "op": "blocks", "fmt": "nvfp4", "matrix": "layer", "M": 8192, "K": 28672, "fill": 0.2},
        # A smaller layer of odd sizes; pairs of blocks share scales where both are there.
        {"name": "blocks_ragged", "op": "blocks", "fmt": "mxfp4", "matrix": "layer", "M": 3056, "K": 8176, "fill": 0.35},
        # Decoding one token with the benchmark's layer.
        {"name": "decode_token", "op": "decode", "fmt": "nvfp4", "dtype": "float16", "matrix": "layer", "M": 8192, "K": 28672, "fill": 0.2, "N": 1},
        # Decoding a batch of 16 sequences.
        {"name": "decode_batch", "op": "decode", "fmt": "mxfp4", "dtype": "bfloat16", "matrix": "layer", "M": 8192, "K": 28672, "fill": 0.2, "N": 16},
        # A smaller layer whose sizes divide nothing, an odd batch.
        {"name": "decode_ragged", "op": "decode", "fmt": "nvfp4", "dtype": "bfloat16", "matrix": "layer", "M": 3056, "K": 8176, "fill": 0.35, "N": 67},
        # A prompt of 4096 tokens through the benchmark's layer (its default workload, in 4 bits).
        {"name": "prefill_prompt", "op": "prefill", "fmt": "nvfp4", "dtype": "float16", "matrix": "layer", "M": 8192, "K": 28672, "fill": 0.2, "N": 4096},
        # A short prompt: few tiles of C, the long axis is split.
        {"name": "prefill_short", "op": "prefill", "fmt": "mxfp4", "dtype": "bfloat16", "matrix": "layer", "M": 4096, "K": 14336, "fill": 0.2, "N": 128},
        # Odd sizes, a batch in between.
        {"name": "prefill_ragged", "op": "prefill", "fmt": "nvfp4", "dtype": "bfloat16", "matrix": "layer", "M": 3056, "K": 8176, "fill": 0.35, "N": 1001},
        # Dense clusters on the diagonal (a layer pruned by blocks of neurons): few steps an output tile, C is most of the traffic.
        {"name": "prefill_clustered", "op": "prefill", "fmt": "mxfp4", "dtype": "float16", "matrix": "clustered", "M": 32768, "K": 32768, "N": 512},
    ]


def _log(rng, lo, hi, multiple):
    """A multiple of `multiple` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi // multiple, max(-(-lo // multiple), round(v / multiple)))) * multiple


def draw(rng):
    c = {"op": rng.choice(["dense", "blocks", "decode", "decode", "prefill", "prefill"]), "fmt": rng.choice(["nvfp4", "mxfp4"])}
    if c["op"] == "dense":
        c["dtype"] = rng.choice(["float16", "bfloat16", "float32"])
        c["N"] = _log(rng, 1, 4096, 1)
        c["K"] = _log(rng, 512, 28672 if c["dtype"] != "float32" else 14336, 16)
        return c
    if c["op"] != "blocks":
        c["dtype"] = rng.choice(["float16", "bfloat16"])
    c["matrix"] = "clustered" if c["op"] == "prefill" and rng.random() < 0.25 else "layer"
    if c["matrix"] == "clustered":
        c["M"] = c["K"] = _log(rng, 2048, 32768, 256)
        c["N"] = _log(rng, 16, 512, 1)
        return c
    c["M"] = _log(rng, 512, 8192, 16)
    c["K"] = _log(rng, 512, 28672, 16)
    c["fill"] = round(rng.uniform(0.05, 0.4), 3)
    c["fill"] = round(min(c["fill"], 8192 * 28672 * 0.2 / (c["M"] * c["K"])), 3)  # stored values of the largest listed layer
    if c["op"] == "decode":
        c["N"] = _log(rng, 1, 128, 1)
    elif c["op"] == "prefill":
        c["N"] = _log(rng, 16, 4096, 1)
    return c


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _blocks_of(case, g):
    """(block-row, block-column) of the stored blocks, ascending."""
    Mb, Kb = case["M"] // 16, case["K"] // 16
    if case["matrix"] == "layer":
        at = torch.randperm(Mb * Kb, generator=g, device="cuda")[:max(1, round(case["fill"] * Mb * Kb))].sort().values
    else:  # clusters of 16 x 16 blocks, shifted a little off the diagonal, and one stray block for every cluster
        n = Mb // 16
        off = torch.randint(-8, 9, (n,), generator=g, device="cuda")
        col = (torch.arange(n, device="cuda") * 16 + off).clamp(0, Kb - 16)
        i = torch.arange(16, device="cuda")
        row = (torch.arange(n, device="cuda") * 16)[:, None, None] + i[None, :, None] + 0 * i[None, None, :]
        at = (row * Kb + col[:, None, None] + i[None, None, :] + 0 * i[None, :, None]).reshape(-1)
        at = torch.cat([at, torch.randint(0, Mb * Kb, (n,), generator=g, device="cuda")]).unique()
    return at // Kb, at % Kb


def _weights(case, g):
    """Stored blocks in fp16 [nnzb][16][16] and their structure."""
    brow, bcol = _blocks_of(case, g)
    rowptr = torch.zeros(case["M"] // 16 + 1, dtype=torch.int32, device="cuda")
    rowptr[1:] = torch.bincount(brow, minlength=case["M"] // 16).cumsum(0)
    vals = torch.randn((brow.numel(), 16, 16), generator=g, device="cuda").mul_(0.02).half()
    return {"brow": brow, "bcol": bcol, "rowptr": rowptr, "vals": vals}


def _acts(case, g):
    """Activations: normal, every token of its own size, and a few outlying channels."""
    x = torch.randn((case["N"], case["K"]), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((case["N"], 1), generator=g, device="cuda"))
    x[:, torch.randint(0, case["K"], (max(1, case["K"] // 512),), generator=g, device="cuda")] *= 16
    return x.to(getattr(torch, case["dtype"]))


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "dense":
        s["x"] = _acts(case, g)
        return s
    w = _weights(case, g)
    if case["op"] == "blocks":
        s["w"] = w
        if own:
            import smat_b200 as S
            s["A"] = S.SparseMatrix.from_bcsr(case["M"], case["K"], w["rowptr"].cpu().numpy(), (w["bcol"] * 16).cpu().numpy(),
                                              w["vals"].reshape(-1).cpu().numpy())
        return s
    s["x"] = _acts(case, g)
    s["w"] = _stored(case, w)
    if own:
        import smat_b200 as S
        A = S.Fp4SparseMatrix.from_codes(case["M"], case["K"], w["rowptr"], (w["bcol"] * 16).int(), s["w"]["codes"], s["w"]["scales"],
                                         fmt=case["fmt"], row_scale=s["w"]["row_scale"])
        s["plan"] = S.Fp4Plan(A)
    return s


def _stored(case, w):
    """The weights as a program has them: codes two to a byte (the even k in the low half), scales, powers of two of the rows."""
    q, scale, p = _quantize_blocks(case, w)
    code = (torch.bucketize(q.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")) + 8 * (q < 0)).to(torch.uint8)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    scales = scale.to(torch.float8_e4m3fn).view(torch.uint8) if case["fmt"] == "nvfp4" else (torch.log2(scale.double()).round() + 127).to(torch.uint8)
    return {"brow": w["brow"], "bcol": w["bcol"], "codes": codes.contiguous(), "scales": scales.contiguous(), "row_scale": p}


# ---- plain forms ----------------------------------------------------------------------------------------------------------------

def _e2m1(q):
    """Nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with the sign of q, ties to the even code, saturating."""
    a = q.abs().clamp(max=6)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((a / step).round() * step, q)


def _pow2_of_rows(amax):
    """Least 2^j >= amax / 2688, j >= -100; 1 for 0."""
    m, e = torch.frexp(amax.float())
    j = e - 12 + (m > 0.65625).int()  # 2688 = 0.65625 * 2^12
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(m), j.clamp(min=-100)), torch.ones_like(m))


def _scale_of(gmax, p, fmt):
    if fmt == "nvfp4":
        return (gmax.double() / 6 / p.double()).float().to(torch.float8_e4m3fn).float()
    e = torch.frexp(gmax.float()).exponent - 3
    return torch.ldexp(torch.ones_like(gmax, dtype=torch.float32), torch.where(gmax > 0, e, -127).clamp(-127, 127))


def _quantize_dense(x, fmt):
    """(codes' values [N][groups][g], scales [N][groups], powers of two [N]); the last group may be cut short (zeros)."""
    g = 16 if fmt == "nvfp4" else 32
    x = x.float()
    p = _pow2_of_rows(x.abs().amax(1)) if fmt == "nvfp4" else None
    if x.shape[1] % g:
        x = torch.nn.functional.pad(x, (0, g - x.shape[1] % g))
    x = x.reshape(x.shape[0], -1, g)
    scale = _scale_of(x.abs().amax(2), 1.0 if p is None else p[:, None], fmt)
    s = scale.double() if p is None else scale.double() * p[:, None]
    q = torch.where(s[..., None] > 0, _e2m1(x.double() / s[..., None]), 0.0).float()  # in 64 bits: the quotient may lie next to a tie
    return q, scale, p


def _quantize_blocks(case, w):
    v = w["vals"].float()
    gmax = v.abs().amax(2)
    p = None
    if case["fmt"] == "nvfp4":
        rows = torch.zeros((case["M"] // 16, 16), device="cuda")
        rows.scatter_reduce_(0, w["brow"][:, None].expand(-1, 16), gmax, "amax")
        p = _pow2_of_rows(rows)
        of_block = p[w["brow"]]
        scale = _scale_of(gmax, of_block, "nvfp4")
        s = scale.double() * of_block
        p = p.reshape(-1)
    else:
        _, pair = torch.unique_consecutive(w["brow"] * case["K"] + w["bcol"] // 2, return_inverse=True)
        both = torch.zeros((int(pair[-1]) + 1, 16), device="cuda")
        both.scatter_reduce_(0, pair[:, None].expand(-1, 16), gmax, "amax")
        scale = _scale_of(both[pair], None, "mxfp4")
        s = scale.double()
    q = torch.where(s[..., None] > 0, _e2m1(v.double() / s[..., None]), 0.0).float()
    return q, scale, p


def _plain_dense(x, fmt):
    q, scale, p = _quantize_dense(x, fmt)
    y = q * (scale if p is None else scale * p[:, None])[..., None]
    return y.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _plain_A(case, w):
    """The weights as a dense fp32 matrix [M][K]."""
    table = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    code = torch.stack([w["codes"] & 15, w["codes"] >> 4], -1).reshape(-1, 16, 16)
    if case["fmt"] == "nvfp4":
        scale = w["scales"].view(torch.float8_e4m3fn).float() * w["row_scale"].reshape(-1, 16)[w["brow"]]
    else:
        scale = torch.ldexp(torch.ones((), device="cuda"), w["scales"].int() - 127)
    A = torch.zeros((case["M"] // 16, case["K"] // 16, 16, 16), device="cuda")
    A[w["brow"], w["bcol"]] = table[code.long()] * scale[..., None]
    return A.permute(0, 2, 1, 3).reshape(case["M"], case["K"])


def run(s):
    case = s["case"]
    if own:
        import smat_b200 as S
        if case["op"] == "dense":
            return {"values": S.Fp4Matrix.quantize(s["x"], fmt=case["fmt"]).dequantize(s["x"].dtype)}
        if case["op"] == "blocks":
            return {"values": S.Fp4SparseMatrix.quantize(s["A"], fmt=case["fmt"]).dequantize().bcsrVal}
        C = torch.empty((case["M"], case["N"]), dtype=s["x"].dtype, device="cuda")
        s["plan"].spmm(s["x"] if case["op"] == "decode" else S.Fp4Matrix.quantize(s["x"], fmt=case["fmt"]), C)
        return {"C": C}
    if case["op"] == "dense":
        return {"values": _plain_dense(s["x"], case["fmt"]).to(s["x"].dtype)}
    if case["op"] == "blocks":
        q, scale, p = _quantize_blocks(case, s["w"])
        if p is not None:
            scale = scale * p.reshape(-1, 16)[s["w"]["brow"]]
        return {"values": (q * scale[..., None]).half().reshape(-1)}
    B = s["x"].float() if case["op"] == "decode" else _plain_dense(s["x"], case["fmt"])
    return {"C": (_plain_A(case, s["w"]) @ B.T).to(s["x"].dtype)}


def work(case):
    size = {"float16": 2, "bfloat16": 2, "float32": 4}.get(case.get("dtype"), 2)
    if case["op"] == "dense":
        return {"bytes": 2 * size * case["N"] * case["K"], "flops": 0}
    if case["matrix"] == "layer":
        nnzb = max(1, round(case["fill"] * (case["M"] // 16) * (case["K"] // 16)))
    else:
        nnzb = case["M"] // 256 * 257
    if case["op"] == "blocks":
        return {"bytes": 2 * 512 * nnzb + 4 * nnzb, "flops": 0}
    A = nnzb * (128 + 16 + 4) + 4 * (case["M"] // 16 + 1) + (4 * case["M"] if case["fmt"] == "nvfp4" else 0)
    return {"bytes": A + 2 * case["N"] * case["K"] + 2 * case["M"] * case["N"], "flops": 512 * nnzb * case["N"]}


# ---- the same from the definition, in 64 bits ---------------------------------------------------------------------------------

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_E4M3 = [m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1]


def _nearest(x, table):
    """Index of the nearest entry of an ascending table; a tie goes to the even index."""
    t = torch.tensor(table, dtype=torch.float64, device=x.device)
    mids = (t[1:] + t[:-1]) / 2
    below, above = torch.bucketize(x, mids), torch.bucketize(x, mids, right=True)
    return torch.where(below % 2 == 0, below, above)


def _exact_quantized(x, group_amax, row_amax, fmt):
    """x [..., k], the largest magnitudes of its group and row [...] -> the values in 4 bits, in 64 bits."""
    if fmt == "nvfp4":
        p = torch.exp2(torch.ceil(torch.log2(row_amax / 2688)))
        p = torch.where(row_amax <= 2688 * p / 2, p / 2, p)  # the logarithm is rounded
        p = torch.where(row_amax > 2688 * p, 2 * p, p).clamp(min=2.0 ** -100)
        p = torch.where(row_amax > 0, p, 1.0)
        s = torch.tensor(_E4M3, dtype=torch.float64, device=x.device)[_nearest(group_amax / (6 * p), _E4M3)] * p
    else:
        e = torch.floor(torch.log2(group_amax))
        e = torch.where(torch.exp2(e) > group_amax, e - 1, torch.where(torch.exp2(e + 1) <= group_amax, e + 1, e)) - 2
        s = torch.exp2(e.clamp(-127, 127))
    s = s[..., None]
    code = _nearest(x.abs() / torch.where(s > 0, s, 1.0), _E2M1)
    v = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)[code] * s
    return torch.where(x < 0, -v, v)


def _exact_dense(x, fmt):
    g = 16 if fmt == "nvfp4" else 32
    x = x.double()
    N, K = x.shape
    groups = -(-K // g)
    full = torch.zeros((N, groups * g), dtype=torch.float64, device=x.device)
    full[:, :K] = x
    full = full.view(N, groups, g)
    rows = full.abs().amax((1, 2))[:, None].expand(N, groups)
    return _exact_quantized(full, full.abs().amax(2), rows, fmt).view(N, -1)[:, :K]


def exact(case, seed):
    g = _gen(seed)
    if case["op"] == "dense":
        return {"values": _exact_dense(_acts(case, g), case["fmt"])}
    w = _weights(case, g)
    Mb, Kb = case["M"] // 16, case["K"] // 16
    if case["op"] == "blocks":
        v = w["vals"].double()
        big = torch.zeros((Mb, Kb + Kb % 2, 16), dtype=torch.float64, device="cuda")  # of every row of every block, absent ones 0
        big[w["brow"], w["bcol"]] = v.abs().amax(2)
        rows = big.amax(1)[w["brow"]]
        if case["fmt"] == "mxfp4":
            big = big.view(Mb, -1, 2, 16).amax(2).repeat_interleave(2, 1)
        return {"values": _exact_quantized(v, big[w["brow"], w["bcol"]], rows, case["fmt"]).reshape(-1)}
    x = _acts(case, g)
    w = _stored(case, w)
    B = x.double() if case["op"] == "decode" else _exact_dense(x, case["fmt"])
    pair = w["codes"].long()
    code = torch.empty((pair.shape[0], 16, 16), dtype=torch.long, device="cuda")
    code[:, :, 0::2], code[:, :, 1::2] = pair % 16, pair // 16
    v = torch.tensor(_E2M1 + [-t for t in _E2M1], dtype=torch.float64, device="cuda")[code]
    if case["fmt"] == "nvfp4":
        t = torch.tensor(_E4M3, dtype=torch.float64, device="cuda")[w["scales"].long()]
        t = t * w["row_scale"].double().view(Mb, 16)[w["brow"]]
    else:
        t = torch.exp2(w["scales"].double() - 127)
    v = v * t[:, :, None]
    C = torch.zeros((Mb, 16, case["N"]), dtype=torch.float64, device="cuda")
    for r in range(0, Mb, 64):  # 64 block-rows at a time
        mine = (w["brow"] >= r) & (w["brow"] < r + 64)
        n = min(64, Mb - r)
        A = torch.zeros((n, 16, case["K"]), dtype=torch.float64, device="cuda").view(n, 16, Kb, 16)
        A[w["brow"][mine] - r, :, w["bcol"][mine]] = v[mine]
        C[r:r + n] = (A.view(n * 16, case["K"]) @ B.T).view(n, 16, -1)
    return {"C": C.view(case["M"], case["N"])}
