"""Cases for the 8-bit block-scaled operators of ``yoda_scheduler_amd.ops.fp8``.

Three operators make one 8-bit linear layer as a language model serves it:

* ``norm``: h = x + residual, y = h / rms(h) * weight, and y in e4m3 with a scale for each 128
  columns of a row (what the next product takes);
* ``quantize``: a matrix in e4m3 with a scale for each 1 x 128 block (activations that no norm
  precedes) or each 128 x 128 block (a weight, when a model is loaded);
* ``matmul``: a (1 x 128 blocks) times the transpose of b (128 x 128 blocks), plus a bias.

The scales are float32 (a block's largest magnitude / 448) or powers of two held in e8m0 (the
smallest power p with the largest magnitude <= 448 p).
"""
import math

import torch

own = False

BLOCK = 128
TOP = 448.0                 # largest e4m3 value
LEAST = 2.0 ** -126         # smallest scale: a smaller block keeps fewer bits
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _case(name, op, rows, cols, inner=0, dtype="bf16", scales="float", residual=False, block_rows=1, bias=False):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "inner": inner, "dtype": dtype, "scales": scales,
            "residual": residual, "block_rows": block_rows, "bias": bias}


def listed():
    return [
        # one token being decoded: latency is all that counts
        _case("norm 1x4096", "norm", 1, 4096, residual=True),
        # a ragged batch on an odd width in fp16, no residual stream
        _case("norm 333x5001 fp16", "norm", 333, 5001, dtype="fp16", scales="pow2"),
        # a long prompt on a wide model
        _case("norm 16384x8192", "norm", 16384, 8192, residual=True, scales="pow2"),
        # a weight on its way into 8 bits when a model is loaded
        _case("quantize 4096x4096 w", "quantize", 4096, 4096, block_rows=128),
        # the wide activations between the two products of a feed-forward layer, of a prompt
        _case("quantize 8191x10240", "quantize", 8191, 10240, scales="pow2"),
        # one token against a square projection
        _case("matmul 1x4096x4096", "matmul", 1, 4096, 4096),
        # a small decoding batch against a wide projection: bound by the weight's bytes
        _case("matmul 16x8192x8192", "matmul", 16, 8192, 8192, scales="pow2"),
        # a decoding batch of a busy server, with a bias
        _case("matmul 128x8192x4096", "matmul", 128, 8192, 4096, bias=True),
        # nothing is a multiple of anything; fp16 out
        _case("matmul 777x5000x1928 fp16", "matmul", 777, 5000, 1928, dtype="fp16", scales="pow2", bias=True),
        # a prompt against a square projection; scales as a checkpoint holds them
        _case("matmul 4096x4096x4096", "matmul", 4096, 4096, 4096),
        # a prompt against a feed-forward projection, hardware scales
        _case("matmul 8192x8192x8192", "matmul", 8192, 8192, 8192, scales="pow2"),
        # a wide projection of a prompt in float scales; fp16 out
        _case("matmul 4096x10240x4096 fp16", "matmul", 4096, 10240, 4096, dtype="fp16"),
    ]


def _spread(rng, low, high):
    """A size spread over its logarithm; half of them odd or ragged, half multiples of 64."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and n >= 64:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["norm", "quantize", "matmul", "matmul"])
    c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "scales": rng.choice(["float", "pow2"]),
         "residual": False, "block_rows": 1, "bias": False, "inner": 0}
    if op == "matmul":
        c["dtype"] = rng.choice(["bf16", "fp16"])         # sums of 8-bit products are handed on in 16 bits
        c["cols"] = _spread(rng, 16, 16384)
        c["inner"] = _spread(rng, 64, 16384)
        c["rows"] = _spread(rng, 1, min(16384, 8192 ** 3 // (c["cols"] * c["inner"])))
        c["bias"] = rng.random() < 0.3
    else:
        c["cols"] = _spread(rng, 64, 16384)
        c["rows"] = _spread(rng, 1, min(16384, 8192 * 8192 // c["cols"]))
        if op == "norm":
            c["residual"] = rng.random() < 0.6
        else:
            c["block_rows"] = rng.choice([1, 128])
    return c


def _blocks(n):
    return -(-n // BLOCK)


def _scale(amax, kind):
    """A block's scale from its largest magnitude; 1 for a block of zeros."""
    if kind == "pow2":
        f, e = torch.frexp(amax)                      # amax = f 2^e, f in [1/2, 1); 448 = 0.875 * 2^9
        p = torch.where(f <= 0.875, e - 9, e - 8).clamp(-126, 127)
        s = ((p + 127) << 23).view(torch.float32)     # 2^p, exactly
    else:
        s = (amax / TOP).clamp_min(LEAST)
    return torch.where(amax > 0, s, torch.ones_like(s))


def _quantize(y, kind, block_rows):
    """float32 y [R, K] -> (e4m3 [R, K padded to blocks], scales [row blocks, K blocks])."""
    r, k = y.shape
    kb, rb = _blocks(k), -(-r // block_rows)
    p = torch.nn.functional.pad(y, (0, kb * BLOCK - k, 0, rb * block_rows - r)).view(rb, block_rows, kb, BLOCK)
    s = _scale(p.abs().amax(dim=(1, 3)), kind)
    q = (p * (1.0 / s)[:, None, :, None]).to(torch.float8_e4m3fn).view(rb * block_rows, kb * BLOCK)[:r]
    return q, s.to(torch.float8_e8m0fnu) if kind == "pow2" else s


def _dequantize(q, s, block_rows):
    """float32 values of a quantized matrix (K padded)."""
    r, k = q.shape
    s = s.float().repeat_interleave(block_rows, 0)[:r]
    return (q.float().view(r, k // BLOCK, BLOCK) * s[:, :, None]).view(r, k)


def _random(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    return g, normal


def prepare(case, seed):
    """The tensors and handles that a serving program holds before the call."""
    _, normal = _random(case, seed)
    t, r, c, k = TYPES[case["dtype"]], case["rows"], case["cols"], case["inner"]
    st = dict(case)
    if case["op"] == "matmul":
        # an activation has a few channels far larger than the rest; a weight keeps its output's size
        x = normal(r, k) * torch.exp(normal(k) * 0.7)
        qa, sa = _quantize(x, case["scales"], 1)
        qb, sb = _quantize(normal(c, k) / math.sqrt(k), case["scales"], BLOCK)
        del x
        # an activation's scales lie block by block, so that the rows of a tile are neighbours
        sa = sa.t().contiguous().t()
        st |= {"qa": qa.contiguous(), "sa": sa, "qb": qb.contiguous(), "sb": sb,
               "bias_t": normal(c).to(t) if case["bias"] else None}
        if own:                               # the handles that the operators before this one return
            from yoda_scheduler_amd.ops import fp8
            st["a"] = fp8.BlockMatrix(st["qa"], st["sa"], cols=k, block_rows=1)
            st["b"] = fp8.BlockMatrix(st["qb"], st["sb"], cols=k, block_rows=BLOCK)
        return st
    st["x"] = (normal(r, c) * torch.exp(normal(c) * 0.7)).to(t)
    if case["op"] == "norm":
        st["weight"] = (1 + 0.1 * normal(c)).to(t)
        st["res"] = (normal(r, c) * 2).to(t) if case["residual"] else None
    return st


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from yoda_scheduler_amd.ops import fp8
    scale_dtype = torch.float8_e8m0fnu if st["scales"] == "pow2" else torch.float32
    if st["op"] == "matmul":
        return {"out": fp8.matmul(st["a"], st["b"], out_dtype=TYPES[st["dtype"]], bias=st["bias_t"])}
    if st["op"] == "quantize":
        q = fp8.quantize(st["x"], block_rows=st["block_rows"], scale_dtype=scale_dtype)
        return {"values": q.values, "scales": q.scales}
    q, h = fp8.add_rms_norm(st["x"], st["weight"], residual=st["res"], eps=EPS, scale_dtype=scale_dtype)
    return {"values": q.values, "scales": q.scales, "residual": h}


def _run_plain(st):
    t = TYPES[st["dtype"]]
    if st["op"] == "matmul":
        out = _dequantize(st["qa"], st["sa"], 1) @ _dequantize(st["qb"], st["sb"], BLOCK).t()
        if st["bias_t"] is not None:
            out = out + st["bias_t"].float()
        return {"out": out.to(t)}
    if st["op"] == "quantize":
        q, s = _quantize(st["x"].float(), st["scales"], st["block_rows"])
        return {"values": q[:, :st["cols"]], "scales": s}
    h = st["x"]
    if st["res"] is not None:
        h = (h.float() + st["res"].float()).to(t)     # the stream is kept in its own type, and the norm reads that
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(1, keepdim=True) + EPS) * st["weight"].float()
    q, s = _quantize(y, st["scales"], 1)
    return {"values": q[:, :st["cols"]], "scales": s, "residual": h if st["res"] is not None else None}


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    one = 1 if case["scales"] == "pow2" else 4
    r, c, k = case["rows"], case["cols"], case["inner"]
    if case["op"] == "matmul":
        scales = one * _blocks(k) * (r + _blocks(c))
        return {"bytes": r * k + c * k + scales + size * (r * c + (c if case["bias"] else 0)), "flops": 2 * r * c * k}
    q = r * c + one * _blocks(c) * -(-r // case["block_rows"])
    if case["op"] == "quantize":
        return {"bytes": r * c * size + q, "flops": 3 * r * c}
    return {"bytes": r * c * size * (3 if case["residual"] else 1) + c * size + q, "flops": 7 * r * c}


def _power(e):
    """2^e in float64, exactly, for whole numbers e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(v):
    """float64 v (|v| <= 464) to the nearest e4m3 value, ties to even: 3 bits after the first, down to steps of 2^-9."""
    _, e = torch.frexp(v)
    step = _power((e - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _exact_blocks(y, kind, block_rows):
    r, k = y.shape
    wide = torch.zeros(-(-r // block_rows) * block_rows, _blocks(k) * BLOCK, dtype=torch.float64, device=y.device)
    wide[:r, :k] = y
    tiles = wide.unfold(0, block_rows, block_rows).unfold(1, BLOCK, BLOCK)
    amax = tiles.abs().amax(dim=(2, 3))
    ratio = amax / TOP
    if kind == "pow2":
        f, e = torch.frexp(ratio)                                # ratio = f 2^e, f in [1/2, 1)
        s = _power(torch.where(f == 0.5, e - 1, e))              # a power of two is its own
    else:
        s = ratio
    s = torch.where(amax > 0, s.clamp_min(LEAST), torch.ones_like(s))
    each = s.repeat_interleave(block_rows, 0)[:r].repeat_interleave(BLOCK, 1)[:, :k]
    return _e4m3(y / each), s


def exact(case, seed):
    """The definition in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "matmul":
        k = case["inner"]

        def full(q, s, rows):
            each = s.double().repeat_interleave(BLOCK, 1)[:, :k]
            return q[:, :k].double() * (each if rows == 1 else each.repeat_interleave(rows, 0)[:q.shape[0]])

        out = torch.mm(full(st["qa"], st["sa"], 1), full(st["qb"], st["sb"], BLOCK).transpose(0, 1).contiguous())
        return {"out": out if st["bias_t"] is None else out + st["bias_t"].double()}
    y = st["x"].double()
    stream = None
    if case["op"] == "norm":
        if st["res"] is not None:
            stream = y + st["res"].double()
            y = stream.to(TYPES[case["dtype"]]).double()         # the definition rounds the stream once
        y = y * st["weight"].double() / torch.sqrt((y * y).sum(1, keepdim=True) / case["cols"] + EPS)
    q, s = _exact_blocks(y, case["scales"], case["block_rows"])
    return {"values": q, "scales": s, "residual": stream} if case["op"] == "norm" else {"values": q, "scales": s}
