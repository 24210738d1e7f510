"""The operators on 4-bit microscaled matrices and on gradients that are timed, as a training or serving loop calls them.

  park     a matrix is quantised and, later, brought back                    (fp4_quantize, fp4_dequantize)
  linear   activations are quantised and multiplied with a packed weight     (fp4_quantize, fp4_matmul)
  dx       gradient of a linear layer's input from its packed weight         (fp4_grad_input)
  dw       gradient of its weight from the packed (parked) activations       (fp4_grad_weight)
  clip     norm of all gradients, and the gradients scaled to at most that   (clip_grad_norm)

Formats: "mx" = MXFP4 (blocks of 32 along a row, scales 2^(byte - 127)), "nv" = NVFP4 (blocks of 16, E4M3 scales and one
scale for the matrix, a power of two).  Weights and parked activations are in hand as packed bytes: a head of 128 bytes
whose first word is the matrix's scale, the codes (rows of 16 bytes for 32 columns, even column in the low nibble), and
from the next multiple of 128 bytes on the scales, in tiles of 128 rows x 4 blocks: row r, block b of a tile
at byte (r % 32) * 16 + (r / 32) * 4 + b.  Sizes are those of the benchmark's matrices (1024, 4096, 5120, 8192, 14336) and ragged ones.
"""
import importlib

import torch

own = False

BLOCK = {"mx": 32, "nv": 16}
METHOD = {"mx": 8, "nv": 9}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one token's activations of a decode step, parked and restored: launches are all there is
        dict(name="park_nv_bf16_1x4096", kind="park", fmt="nv", dtype="bf16", rows=1, cols=4096),
        # a ragged FP32 matrix: rows that end inside a block and start off any alignment wider than 8 bytes
        dict(name="park_mx_f32_3673x5182", kind="park", fmt="mx", dtype="f32", rows=3673, cols=5182),
        # the MLP activations of a layer, parked between forward and backward
        dict(name="park_nv_bf16_4096x14336", kind="park", fmt="nv", dtype="bf16", rows=4096, cols=14336),
        # a decode step's MLP product for one token: the weight's bytes are all there is
        dict(name="linear_nv_bf16_1x4096x14336", kind="linear", fmt="nv", dtype="bf16", rows=1, cols=4096, out=14336),
        # ragged rows and outputs, FP16 activations
        dict(name="linear_mx_f16_777x5120x1031", kind="linear", fmt="mx", dtype="f16", rows=777, cols=5120, out=1031),
        # a training step's MLP product
        dict(name="linear_nv_bf16_4096x4096x14336", kind="linear", fmt="nv", dtype="bf16", rows=4096, cols=4096, out=14336),
        # a few tokens' input gradient (tuning on short prompts): the weight's bytes again
        dict(name="dx_mx_16x4096x14336", kind="dx", fmt="mx", dtype="bf16", rows=16, cols=14336, out=4096),
        # the MLP's input gradient of a training step
        dict(name="dx_nv_4096x14336x4096", kind="dx", fmt="nv", dtype="bf16", rows=4096, cols=4096, out=14336),
        # ragged tokens, outputs and columns: rows of dY off 16 bytes
        dict(name="dw_mx_1501x1031x3001", kind="dw", fmt="mx", dtype="bf16", rows=1501, cols=3001, out=1031),
        # the MLP's weight gradient of a training step, in FP32 as an optimiser takes it
        dict(name="dw_nv_f32_4096x4096x14336", kind="dw", fmt="nv", dtype="f32", rows=4096, cols=14336, out=4096),
        # the gradients of rank-64 factors of a few layers
        dict(name="clip_f32_24_small", kind="clip", dtype="f32", count=24, rows=64, cols=1024, max_norm=1.0, scale=0.01),
        # the gradients of a layer: attention and MLP matrices and the vectors between them
        dict(name="clip_bf16_14_large", kind="clip", dtype="bf16", count=14, rows=4096, cols=8192, max_norm=1.0, scale=0.001),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["park", "linear", "dx", "dw", "clip"])
    if kind == "clip":
        rows, cols = _log(rng, 1, 4096), _log(rng, 16, 8192)
        return dict(kind=kind, dtype=rng.choice(["f32", "bf16", "f16"]), count=rng.randint(2, 14), rows=rows, cols=cols,
                    max_norm=rng.choice([0.5, 1.0, 1e4]), scale=0.001 * 10 ** (2 * rng.random()))
    case = dict(kind=kind, fmt=rng.choice(["mx", "nv"]), dtype=rng.choice(["f32", "bf16", "f16"]), rows=_log(rng, 1, 4096), cols=_log(rng, 33, 14336))
    if kind == "park":
        return case
    if kind != "linear":
        case["dtype"] = rng.choice(["bf16", "f32"])
    case["out"] = _log(rng, 16, 4096)
    return case


# ---- the plain form -----------------------------------------------------------------------------------------------

def _pow2(e):
    return torch.ldexp(torch.ones((), device=e.device), e)


def _e2m1(x, s):
    """Codes of x / s to nearest, ties to even: the halfway points times s are exact in 32 bits."""
    a = x.abs()
    code = torch.zeros_like(a)
    for mid, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= mid * s) if up else (a > mid * s)
    code = torch.where(s > 0, code, torch.zeros_like(code))
    return code.to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)


def _levels(device):
    m = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)
    return torch.cat([m, -m])


def _quantize(x, fmt):
    """(codes, scale bytes, matrix scale) of a 2-D matrix; the last block of a row is filled up with zeros."""
    rows, cols = x.shape
    bs = BLOCK[fmt]
    blocks = -(-cols // bs)
    v = torch.zeros((rows, blocks * bs), device=x.device)
    v[:, :cols] = x.float()
    v = v.view(rows, blocks, bs)
    bad = ~torch.isfinite(v).all(dim=2)
    v = torch.where(bad[..., None], torch.zeros_like(v), v)
    amax = v.abs().amax(dim=2)
    if fmt == "mx":
        g = torch.ones((), device=x.device)
        e = (torch.frexp(amax)[1] - 3).clamp(-127, 125)
        e = torch.where(amax > 0, e, torch.full_like(e, -127))
        byte = torch.where(bad, torch.full_like(e, 255), e + 127)
        half = torch.div(e, 2, rounding_mode="floor")
        w = v * _pow2(-half)[..., None] * _pow2(half - e)[..., None]
        codes = _e2m1(w, torch.ones_like(w))
    else:
        top = x.float()
        top = torch.where(torch.isfinite(top), top, torch.zeros_like(top)).abs().max()
        m, e = torch.frexp(top)
        t = (e - 12 + (m > 0.65625)).clamp(-110, 117)
        g = _pow2(torch.where(top > 0, t, torch.zeros_like(t)))
        inv = 1 / g
        s8 = (amax * inv / 6).clamp(max=448.0).to(torch.float8_e4m3fn)
        byte = torch.where(bad, torch.full(bad.shape, 0x7F, dtype=torch.uint8, device=x.device), s8.view(torch.uint8))
        codes = _e2m1(v * inv, s8.float()[..., None])
    return codes.view(rows, -1), byte.to(torch.uint8), g


def _scale_values(byte, fmt):
    if fmt == "nv":
        return byte.view(torch.float8_e4m3fn).float()
    e = byte.to(torch.int32) - 127
    half = torch.div(e, 2, rounding_mode="floor")
    return torch.where(e == 128, torch.full(e.shape, float("nan"), device=e.device), _pow2(half) * _pow2(e - half))


def _values(codes, byte, g, fmt, cols):
    rows = codes.shape[0]
    v = _levels(codes.device)[codes.long()].view(rows, -1, BLOCK[fmt]) * _scale_values(byte, fmt)[..., None] * g
    return v.view(rows, -1)[:, :cols]


def _sizes(rows, cols, fmt):
    ld = -(-cols // 32) * 16
    at = -(-(128 + rows * ld) // 128) * 128
    groups, quads = -(-rows // 128), -(-(-(-cols // BLOCK[fmt])) // 4)
    return ld, at, groups, quads


def _pack(codes, byte, g, fmt, cols):
    rows, blocks = byte.shape
    ld, at, groups, quads = _sizes(rows, cols, fmt)
    out = torch.zeros(at + groups * quads * 512, dtype=torch.uint8, device=codes.device)
    out[:4] = g.float().reshape(1).view(torch.uint8)
    wide = torch.zeros((rows, 2 * ld), dtype=torch.uint8, device=codes.device)
    wide[:, : codes.shape[1]] = codes
    out[128: 128 + rows * ld] = (wide[:, 0::2] | (wide[:, 1::2] << 4)).reshape(-1)
    full = torch.zeros((groups * 128, quads * 4), dtype=torch.uint8, device=codes.device)
    full[:rows, :blocks] = byte
    out[at:] = full.view(groups, 4, 32, quads, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    return out


def _unpack(data, rows, cols, fmt):
    """(codes, scale bytes, matrix scale) of packed bytes."""
    ld, at, groups, quads = _sizes(rows, cols, fmt)
    g = data[:4].view(torch.float32)[0]
    pairs = data[128: 128 + rows * ld].view(rows, ld)
    blocks = -(-cols // BLOCK[fmt])
    codes = torch.stack([pairs & 15, pairs >> 4], dim=2).view(rows, -1)[:, : blocks * BLOCK[fmt]]
    full = data[at:].view(groups, quads, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(groups * 128, quads * 4)
    return codes.contiguous(), full[:rows, :blocks].contiguous(), g


def _plain(state):
    c = state["case"]
    if c["kind"] == "clip":
        total = torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt()
        coef = (c["max_norm"] / (total + EPS)).clamp(max=1.0).float()
        return {"norm": total.float(), "grads": [(g.float() * coef).to(g.dtype) for g in state["grads"]]}
    if c["kind"] == "park":
        return _values(*_quantize(state["x"], c["fmt"]), c["fmt"], c["cols"]).to(state["x"].dtype)
    if c["kind"] == "linear":
        x = _values(*_quantize(state["x"], c["fmt"]), c["fmt"], c["cols"])
        w = _values(*_unpack(state["w"], c["out"], c["cols"], c["fmt"]), c["fmt"], c["cols"])
        return (x @ w.t()).to(torch.bfloat16)
    dy = state["dy"].float()
    if c["kind"] == "dx":
        w = _values(*_unpack(state["w"], c["out"], c["cols"], c["fmt"]), c["fmt"], c["cols"])
        return (dy @ w).to(DTYPE[c["dtype"]])
    x = _values(*_unpack(state["x4"], c["rows"], c["cols"], c["fmt"]), c["fmt"], c["cols"])
    return (dy.t() @ x).to(DTYPE[c["dtype"]])


# ---- what a user's program does ------------------------------------------------------------------------------------

def _ours(state):
    ops = importlib.import_module("bitsqueeze-llm_b200.torch_ops")
    c = state["case"]
    if c["kind"] == "clip":
        norm = ops.clip_grad_norm(state["grads"], c["max_norm"], out=state["outs"])
        return {"norm": norm, "grads": state["outs"]}
    method = METHOD[c["fmt"]]
    if c["kind"] == "park":
        return ops.fp4_dequantize(ops.fp4_quantize(state["x"], method), state["x"].dtype)
    if c["kind"] == "linear":
        w = ops.Fp4Matrix(state["w"], c["out"], c["cols"], method)
        return ops.fp4_matmul(ops.fp4_quantize(state["x"], method), w, torch.bfloat16)
    if c["kind"] == "dx":
        return ops.fp4_grad_input(state["dy"], ops.Fp4Matrix(state["w"], c["out"], c["cols"], method), DTYPE[c["dtype"]])
    return ops.fp4_grad_weight(state["dy"], ops.Fp4Matrix(state["x4"], c["rows"], c["cols"], method), DTYPE[c["dtype"]])


def run(state):
    return _ours(state) if own else _plain(state)


def _shapes(c):
    """A matrix, a vector, a smaller ragged matrix, in turn."""
    full = [(c["rows"], c["cols"]), (c["cols"],), (c["rows"] // 2 + 1, c["cols"] // 2 + 1)]
    return [full[i % 3] for i in range(c["count"])]


def _activations(gen, rows, cols, dtype):
    """N(0, 1) with a few columns scaled up, as a layer's activations are."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    n = max(1, cols // 1000)
    at = torch.randperm(cols, generator=gen, device="cuda")[:n]
    x[:, at] *= 20 + 80 * torch.rand(n, generator=gen, device="cuda")
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    kind = case["kind"]
    if kind == "clip":
        state["grads"] = [(torch.randn(s, generator=gen, device="cuda") * case["scale"]).to(DTYPE[case["dtype"]]) for s in _shapes(case)]
        state["outs"] = [torch.empty_like(g) for g in state["grads"]]
        return state
    rows, cols = case["rows"], case["cols"]
    if kind in ("park", "linear"):
        state["x"] = _activations(gen, rows, cols, DTYPE[case["dtype"]])
    if kind in ("linear", "dx"):
        w = torch.randn((case["out"], cols), generator=gen, device="cuda") * 0.02
        state["w"] = _pack(*_quantize(w, case["fmt"]), case["fmt"], cols)
    if kind in ("dx", "dw"):
        state["dy"] = (torch.randn((rows, case["out"]), generator=gen, device="cuda") * 1e-3).to(torch.bfloat16)
    if kind == "dw":
        x = _activations(gen, rows, cols, torch.bfloat16)
        state["x4"] = _pack(*_quantize(x, case["fmt"]), case["fmt"], cols)
    return state


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if case["kind"] == "clip":
        n = sum(s[0] * (s[1] if len(s) > 1 else 1) for s in _shapes(case))
        return {"bytes": 2 * n * size + 4, "flops": 3 * n}
    rows, cols = case["rows"], case["cols"]
    four = 0.5 + 1 / BLOCK[case["fmt"]]
    if case["kind"] == "park":
        return {"bytes": rows * cols * 2 * size, "flops": 3 * rows * cols}
    flops = 2 * rows * cols * case["out"]
    if case["kind"] == "linear":
        return {"bytes": rows * cols * size + case["out"] * cols * four + 2 * rows * case["out"], "flops": flops}
    if case["kind"] == "dx":
        return {"bytes": 2 * rows * case["out"] + case["out"] * cols * four + rows * cols * size, "flops": flops}
    return {"bytes": 2 * rows * case["out"] + rows * cols * four + case["out"] * cols * size, "flops": flops}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def _nearest(a, table):
    """Index of the nearest entry of an ascending table, a tie to the even index (its code has a mantissa that ends in 0)."""
    mids = (table[1:] + table[:-1]) / 2
    up = torch.bucketize(a, mids, right=False)          # first i with mids[i] >= a: entries below a's interval
    tie = (up < mids.numel()) & (mids[up.clamp(max=mids.numel() - 1)] == a)
    return torch.where(tie & (up % 2 == 1), up + 1, up)


def _exact_values(x, fmt):
    """What a finite matrix holds after quantisation, from the formulas, in 64 bits."""
    rows, cols = x.shape
    bs = BLOCK[fmt]
    v = torch.nn.functional.pad(x.double(), (0, -cols % bs)).view(rows, -1, bs)
    amax = v.abs().amax(dim=2, keepdim=True)
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    if fmt == "mx":
        s = torch.ldexp(torch.ones_like(amax), (torch.frexp(amax)[1] - 3).clamp(min=-127))
    else:
        top = x.double().abs().max()
        m, e = torch.frexp(top / 2688)
        t = torch.where(m > 0.5, e, e - 1).clamp(min=-110)
        g = torch.ldexp(torch.ones_like(top), torch.where(top > 0, t, torch.zeros_like(t)))
        e4m3 = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
        s = e4m3[_nearest((amax / (6 * g)).contiguous(), e4m3)] * g
    q = torch.where(s > 0, v.abs() / s, torch.zeros_like(v))
    out = torch.where(v < 0, -1.0, 1.0) * levels[_nearest(q.contiguous(), levels)] * s
    return out.view(rows, -1)[:, :cols]


def _exact_unpacked(data, rows, cols, fmt):
    codes, byte, g = _unpack(data, rows, cols, fmt)
    s = byte.view(torch.float8_e4m3fn).double() if fmt == "nv" else torch.exp2(byte.double() - 127)
    m = (codes & 7).double()
    mag = torch.where(m < 2, m / 2, torch.exp2(torch.floor(m / 2) - 1) * (1 + (m % 2) / 2))
    v = torch.where(codes > 7, -mag, mag).view(rows, -1, BLOCK[fmt]) * s[..., None] * g.double()
    return v.view(rows, -1)[:, :cols]


def exact(case, seed):
    state = prepare(case, seed)
    kind, fmt, rows, cols = case["kind"], case.get("fmt"), case["rows"], case["cols"]
    if kind == "clip":
        flat = [g.double() for g in state["grads"]]
        norm = torch.sqrt(sum((g * g).sum() for g in flat))
        coef = min(1.0, case["max_norm"] / (float(norm) + EPS))
        return {"norm": norm, "grads": [g * coef for g in flat]}
    if kind == "park":
        return _exact_values(state["x"], fmt)
    if kind == "linear":
        return _exact_values(state["x"], fmt) @ _exact_unpacked(state["w"], case["out"], cols, fmt).t()
    if kind == "dx":
        return state["dy"].double() @ _exact_unpacked(state["w"], case["out"], cols, fmt)
    return state["dy"].double().t() @ _exact_unpacked(state["x4"], rows, cols, fmt)
