"""Cases and plain forms of the block-scaled FP8 operators: what a linear layer in e4m3 calls.

The product C = A * B^T with one power-of-two scale for each block of 128 values, the quantiser
that makes its operands, the root-mean-square norm that produces the left operand directly, and
that norm's backward pass.  `own = False` computes each operator in elementary torch operations
in 32 bits; `own = True` calls the library.

A scale is one byte s (E8M0) that stands for 2^(s - 127).  For a block of values with the largest
finite magnitude a > 0 it is the smallest power of two with a / 2^(s - 127) <= 448, the largest
e4m3 value; for a block of zeros it stands for 1.  A value x of the block is held as
e4m3(x / 2^(s - 127)), rounded to nearest even.
"""

import ctypes

import torch

own = False

BF16, F32 = 0, 1  # the library's numbers for the two types
TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
NUMBER = {"bf16": BF16, "f32": F32}
EPS = 1e-5


def up(n, to):
    return -(-n // to) * to


# --------------------------------------------------------------------- cases


def listed():
    return [
        # one token through a square projection: the weights are read once, nothing else counts
        dict(name="gemm token", op="gemm", m=1, n=8192, k=8192, block_b=128, c="bf16"),
        # the smallest call: a decode step's narrow projection, where the launch counts
        dict(name="gemm token narrow", op="gemm", m=1, n=1024, k=2048, block_b=128, c="bf16"),
        # a decode batch that fills no tile
        dict(name="gemm batch 48", op="gemm", m=48, n=4096, k=8192, block_b=128, c="bf16"),
        # a ragged prompt: no size is a multiple of a tile or of 128
        dict(name="gemm ragged prompt", op="gemm", m=1000, n=4600, k=2064, block_b=128, c="bf16"),
        # the library's own headline size
        dict(name="gemm 8192", op="gemm", m=8192, n=8192, k=8192, block_b=128, c="bf16"),
        # a weight gradient dY^T X: both operands scaled by row, fp32 out, tokens along K
        dict(name="gemm weight gradient", op="gemm", m=4096, n=8192, k=4096, block_b=1, c="f32"),
        # one token's activation
        dict(name="quantize token", op="quantize", rows=1, cols=8192, block=1, both=False, type="bf16"),
        # a training step's activation gradient: rows for the input's gradient, columns for the weights'
        dict(name="quantize both ways", op="quantize", rows=8192, cols=8192, block=1, both=True, type="bf16"),
        # one token through the norm before a projection
        dict(name="norm token", op="norm", rows=1, cols=8192, residual=True, train=False, type="bf16"),
        # a prompt's norms
        dict(name="norm 8192", op="norm", rows=8192, cols=8192, residual=True, train=False, type="bf16"),
        # gradients of a short ragged batch of an odd width
        dict(name="norm backward ragged", op="norm_backward", rows=1000, cols=4600, residual=True, type="bf16"),
        # gradients of a full batch
        dict(name="norm backward 8192", op="norm_backward", rows=8192, cols=8192, residual=True, type="bf16"),
    ]


def spread(rng, low, high):
    """A whole number, even over its logarithm."""
    return min(high, int(low * (high / low) ** rng.random() + 0.5))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "quantize", "norm", "norm_backward"])
    if op == "gemm":
        return dict(op=op, m=spread(rng, 1, 8192), n=spread(rng, 64, 8192), k=spread(rng, 64, 8192),
                    block_b=rng.choice([1, 128]), c=rng.choice(["bf16", "f32"]))
    rows, cols = spread(rng, 1, 8192), spread(rng, 64, 8192)
    kind = rng.choice(["bf16", "bf16", "f32"])
    if op == "quantize":
        return dict(op=op, rows=rows, cols=cols, block=rng.choice([1, 128]),
                    both=rng.choice([False, True]), type=kind)
    if op == "norm":
        return dict(op=op, rows=rows, cols=cols, residual=rng.choice([False, True]),
                    train=rng.choice([False, True]), type=kind)
    return dict(op=op, rows=rows, cols=cols, residual=rng.choice([False, True]), type=kind)


def work(case):
    c = case
    if c["op"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        groups = up(k, 128) // 128
        out = 2 if c["c"] == "bf16" else 4
        scales = (m + (n if c["block_b"] == 1 else up(n, 128) // 128)) * groups
        return {"bytes": m * k + n * k + scales + m * n * out, "flops": 2 * m * n * k}
    rows, cols = c["rows"], c["cols"]
    size, n = (2 if c["type"] == "bf16" else 4), rows * cols
    per_row = rows * (up(cols, 128) // 128)
    if c["op"] == "quantize":
        each = n + (per_row if c["block"] == 1 else per_row // 128)
        return {"bytes": n * size + each * (2 if c["both"] else 1), "flops": 3 * n}
    if c["op"] == "norm":
        read = n * size * (2 if c["residual"] else 1) + cols * 2
        write = n + per_row + (n * size if c["residual"] else 0)
        if c["train"]:
            write += n * size + rows * 4
        return {"bytes": read + write, "flops": 7 * n}
    return {"bytes": n * size * (4 if c["residual"] else 3) + cols * 6 + rows * 4, "flops": 10 * n}


# -------------------------------------------------------------------- inputs


def values(gen, rows, cols, scale=1.0):
    """Activations as they come: normal, with columns of quite different size."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= torch.exp(torch.randn(cols, generator=gen, device="cuda")) * scale
    return x


def bytes_for(rows, cols):
    """Room for rows x cols bytes, each row at a multiple of 16."""
    return torch.zeros(rows, up(cols, 16), dtype=torch.uint8, device="cuda")


def padded(q):
    out = bytes_for(*q.shape)
    out[:, :q.shape[1]] = q
    return out


def ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        qa, sa = quantized(values(gen, m, k), 1)
        w = values(gen, n, k, k ** -0.5)
        qb, sb = quantized(w, case["block_b"])
        s["a"], s["sa"], s["b"], s["sb"] = (padded(t) for t in (qa, sa, qb, sb))
        s["out"] = torch.zeros(m, n, dtype=TYPE[case["c"]], device="cuda")
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return s
    rows, cols, t = case["rows"], case["cols"], TYPE[case["type"]]
    groups, groups_t = up(cols, 128) // 128, up(rows, 128) // 128
    s["x"] = values(gen, rows, cols).to(t)
    if case["op"] == "quantize":
        tall = 1 if case["block"] == 1 else 128
        s["q"] = bytes_for(rows, cols)
        s["s"] = bytes_for(up(rows, tall) // tall, groups)
        if case["both"]:
            s["qt"] = bytes_for(cols, rows)
            s["st"] = bytes_for(up(cols, tall) // tall, groups_t)
        return s
    s["w"] = (1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(torch.bfloat16)
    s["r"] = (3 * torch.randn(rows, cols, generator=gen, device="cuda")).to(t)
    if case["op"] == "norm":
        s["h"] = torch.zeros(rows, cols, dtype=t, device="cuda")
        s["y"] = torch.zeros(rows, cols, dtype=t, device="cuda")
        s["q"], s["s"] = bytes_for(rows, cols), bytes_for(rows, groups)
        s["rstd"] = torch.zeros(rows, device="cuda")
        return s
    # what the forward pass left behind, the gradient of its output and the residual's own
    s["h"] = s.pop("r")
    s["rstd"] = torch.rsqrt(s["h"].float().square().mean(dim=1) + EPS)
    s["dy"] = s.pop("x")
    s["dh"] = torch.randn(rows, cols, generator=gen, device="cuda").to(t)
    s["dx"] = torch.zeros(rows, cols, dtype=t, device="cuda")
    s["dw"] = torch.zeros(cols, device="cuda")
    s["room"] = torch.zeros(room_for(rows, cols), dtype=torch.uint8, device="cuda")
    return s


def room_for(rows, cols):
    """A workspace that is large enough on any device: the library asks for at most 1024 partial
    rows of 32-bit sums (cmb_rmsnorm_backward_workspace_bytes says how much it needs)."""
    return 4 * up(cols, 64) * min(rows, 1024) + 256


# ---------------------------------------------------------------- plain forms


def quantized(x, block):
    """x (32 bits) as e4m3 bytes and E8M0 bytes: one scale for 128 values of a row (block 1), or
    for a block of 128 x 128 (block 128)."""
    rows, cols = x.shape
    full = torch.zeros(up(rows, block), up(cols, 128), device=x.device)
    full[:rows, :cols] = x
    tiles = full.view(full.shape[0] // block, block, full.shape[1] // 128, 128)
    top = tiles.abs().amax(dim=(1, 3))
    m, e = torch.frexp(top)  # top = m * 2^e with m in [0.5, 1), and 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).int()
    e = torch.where(top > 0, e.clamp(min=-127), torch.zeros_like(e))
    q = torch.ldexp(tiles, -e[:, None, :, None]).reshape(full.shape)[:rows, :cols]
    return q.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def restored(q, s, cols, block):
    """The 32-bit values that e4m3 bytes and their scales stand for."""
    rows = q.shape[0]
    x = q[:, :cols].contiguous().view(torch.float8_e4m3fn).float()
    e = s[:, :up(cols, 128) // 128].int() - 127
    e = e.repeat_interleave(128, dim=1)[:, :cols].repeat_interleave(block, dim=0)[:rows]
    return torch.ldexp(x, e)


def e4m3(q, cols):
    return q[:, :cols].view(torch.float8_e4m3fn)


def e8m0(s, cols):
    return s[:, :up(cols, 128) // 128].view(torch.float8_e8m0fnu)


def run(state):
    return {"gemm": run_gemm, "quantize": run_quantize, "norm": run_norm,
            "norm_backward": run_norm_backward}[state["op"]](state)


def run_gemm(s):
    if own:
        from cuda_micro_bench_b200 import check

        a, sa, b, sb, out = s["a"], s["sa"], s["b"], s["sb"], s["out"]
        check("cmb_gemm_e4m3_block128", ptr(a), a.shape[1], ptr(sa), sa.shape[1], ptr(b),
              b.shape[1], ptr(sb), sb.shape[1], s["block_b"], ptr(out), out.shape[1],
              NUMBER[s["c"]], s["m"], s["n"], s["k"], ptr(s["status"]), stream())
        return out
    a = restored(s["a"], s["sa"], s["k"], 1)
    b = restored(s["b"], s["sb"], s["k"], s["block_b"])
    return (a @ b.t()).to(TYPE[s["c"]])


def run_quantize(s):
    rows, cols = s["rows"], s["cols"]
    if own:
        from cuda_micro_bench_b200 import check

        x, q, sc = s["x"], s["q"], s["s"]
        back = [ptr(s["qt"]), s["qt"].shape[1], ptr(s["st"]), s["st"].shape[1]] if s["both"] else [
            None, 0, None, 0]
        check("cmb_quantize_e4m3_block128", ptr(x), NUMBER[s["type"]], rows, cols, x.shape[1],
              s["block"], ptr(q), q.shape[1], ptr(sc), sc.shape[1], *back, stream())
        out = [e4m3(q, cols), e8m0(sc, cols)]
        return out + ([e4m3(s["qt"], rows), e8m0(s["st"], rows)] if s["both"] else [])
    x = s["x"].float()
    out = list(quantized(x, s["block"]))
    if s["both"]:
        out += quantized(x.t(), s["block"])
    return [t.view(torch.float8_e8m0fnu if i % 2 else torch.float8_e4m3fn)
            for i, t in enumerate(out)]


def run_norm(s):
    rows, cols = s["rows"], s["cols"]
    if own:
        from cuda_micro_bench_b200 import check

        x, q, sc, kind = s["x"], s["q"], s["s"], NUMBER[s["type"]]
        r, h = (ptr(s["r"]), ptr(s["h"])) if s["residual"] else (None, None)
        y, rstd = (ptr(s["y"]), ptr(s["rstd"])) if s["train"] else (None, None)
        check("cmb_rmsnorm_e4m3_block128", ptr(x), cols, r, cols, kind, ptr(s["w"]), BF16,
              ctypes.c_float(EPS), rows, cols, h, cols, y, cols, ptr(q), q.shape[1], ptr(sc),
              sc.shape[1], rstd, stream())
        out = {"q": e4m3(q, cols), "s": e8m0(sc, cols)}
        if s["residual"]:
            out["h"] = s["h"]
        if s["train"]:
            out.update(y=s["y"], rstd=s["rstd"])
        return out
    h = (s["x"].float() + s["r"].float()).to(TYPE[s["type"]]) if s["residual"] else s["x"]
    rstd = torch.rsqrt(h.float().square().mean(dim=1) + EPS)
    y = h.float() * rstd[:, None] * s["w"].float()
    q, sc = quantized(y, 1)
    out = {"q": q.view(torch.float8_e4m3fn), "s": sc.view(torch.float8_e8m0fnu)}
    if s["residual"]:
        out["h"] = h
    if s["train"]:
        out.update(y=y.to(TYPE[s["type"]]), rstd=rstd)
    return out


def run_norm_backward(s):
    rows, cols = s["rows"], s["cols"]
    if own:
        from cuda_micro_bench_b200 import check

        dh = ptr(s["dh"]) if s["residual"] else None
        check("cmb_rmsnorm_backward", ptr(s["dy"]), cols, ptr(s["h"]), cols, dh, cols,
              NUMBER[s["type"]], ptr(s["w"]), BF16, ptr(s["rstd"]), rows, cols, ptr(s["dx"]), cols,
              ptr(s["dw"]), ptr(s["room"]), s["room"].numel(), stream())
        return {"dx": s["dx"], "dw": s["dw"]}
    dy, unit = s["dy"].float(), s["h"].float() * s["rstd"][:, None]
    g = dy * s["w"].float()
    dx = s["rstd"][:, None] * (g - unit * (g * unit).mean(dim=1, keepdim=True))
    if s["residual"]:
        dx = dx + s["dh"].float()
    # long sums over the rows: in 64 bits, rounded once
    return {"dx": dx.to(TYPE[s["type"]]), "dw": (dy * unit).double().sum(dim=0).float()}


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


# --------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "gemm":
        return whole(s["a"], s["sa"], s["k"], 1) @ whole(s["b"], s["sb"], s["k"], s["block_b"]).T
    if s["op"] == "quantize":
        out = list(scaled(s["x"].double(), s["block"]))
        return out + (list(scaled(s["x"].double().T, s["block"])) if s["both"] else [])
    if s["op"] == "norm":
        h = s["x"].double()
        if s["residual"]:
            h = (h + s["r"].double()).to(s["x"].dtype).double()  # h is held in the inputs' type
        rstd = (h.pow(2).sum(1) / s["cols"] + EPS).pow(-0.5)
        y = h * rstd.unsqueeze(1) * s["w"].double()
        out = dict(zip(("q", "s"), scaled(y, 1)))
        if s["residual"]:
            out["h"] = h
        if s["train"]:
            out["y"], out["rstd"] = y, rstd
        return out
    # y_j = w_j h_j r with r = (sum h^2 / D + eps)^-1/2, so dr/dh_i = -r^3 h_i / D
    dy, h, w, r = (s[n].double() for n in ("dy", "h", "w", "rstd"))
    r = r.unsqueeze(1)
    along = (dy * w * h).sum(1, keepdim=True)
    dx = dy * w * r - r.pow(3) * h * along / s["cols"]
    return {"dx": dx + s["dh"].double() if s["residual"] else dx, "dw": (dy * h * r).sum(0)}


def whole(q, s, cols, block):
    """What bytes and scales stand for, by the place of each value."""
    col = torch.arange(cols, device=q.device)
    row = torch.arange(q.shape[0], device=q.device)
    two = torch.exp2(s.double() - 127)[row // block][:, col // 128]
    return q.view(torch.float8_e4m3fn)[:, :cols].double() * two


def scaled(x, block):
    """x / scale before its rounding to e4m3, and the scales, by blocks found one edge at a time."""
    rows, cols = x.shape
    high, wide = up(rows, block) // block, up(cols, 128) // 128
    big = x.abs()
    big = torch.nn.functional.pad(big, (0, wide * 128 - cols, 0, high * block - rows))
    big = big.unflatten(1, (wide, 128)).amax(2).unflatten(0, (high, block)).amax(1)
    # the smallest power of two that is not under big / 448, between 2^-127 and 2^127
    e = torch.ceil(torch.log2(big / 448))
    e = torch.where(torch.exp2(e - 1) * 448 >= big, e - 1, e)
    e = torch.where(torch.exp2(e) * 448 < big, e + 1, e)
    two = torch.where(big > 0, torch.exp2(e.clamp(-127, 127)), torch.ones_like(big))
    row = torch.arange(rows, device=x.device) // block
    col = torch.arange(cols, device=x.device) // 128
    return x / two[row][:, col], two
