"""Products in microscaled 4-bit floating point: what is measured of them, their plain forms and their definition in 64 bits.

The format.  A row of K values is cut into blocks of 32.  A block has one scale, a power of two 2^(b - 127) held as the byte
b (255 stands for NaN), and every value is held in four bits as a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, times the scale.
Rounding a block: the scale is the smallest power of two X with max|x| <= 7 X (a value of up to 7 X is as near to 6 X as a step
of the coarser scale would bring it), each x / X goes to the nearest of the eight, ties to the even code, and to 6 beyond.

    codes   uint8 [R, 16 ceil(K / 32)]   value 2 i in the low half of byte i, value 2 i + 1 in the high half; zeros beyond K
    scales  uint8 [ceil(R / 128), ceil(K / 128), 512]   the byte of row r, block j in tile (r / 128, j / 4) at
            16 (r % 32) + 4 ((r % 128) / 32) + j % 4

Three kinds of case:

``quantise``      rows of activations or weights into that form, and the values that they then stand for.
``product``       y[T, N] = x[T, K] w[N, K]^T of two matrices in that form, as a projection whose input is there already.
``feed_forward``  a gated feed-forward behind its norm, as a decoder layer runs it:
                      s   <- s + d                                  (float32 residual stream, the sub-layer before it)
                      h   <- quantise(s / sqrt(mean(s^2) + eps) * g)
                      a   <- quantise(silu(gate) * up),  gate and up: the products of h with rows of the merged weight, whose
                             rows alternate in blocks of eight (eight of the gate, eight of the up projection)
                      y   <- a w_down^T
                  and it returns the stream and y.

Widths are those of the layer sizes that the benchmark and the tests of this repository name (width 4,096 with 12,288, width
5,120 with 25,600, width 1,024) and of its smaller test models, beside odd ones.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
TILE_ROWS, TILE_BLOCKS = 128, 4
EPS = 1e-6
DT = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one token's row of the widest layer here, on its way into the down projection: the smallest call
        {"name": "quantise_1x12288", "kind": "quantise", "rows": 1, "width": 12288, "pitch": 12288, "dtype": "bfloat16"},
        # an odd number of rows that are columns of a wider buffer, a last block that is not full, float32 activations
        {"name": "quantise_333x1000_f32", "kind": "quantise", "rows": 333, "width": 1000, "pitch": 1500, "dtype": "float32"},
        # a weight as it is loaded
        {"name": "quantise_24576x4096", "kind": "quantise", "rows": 24576, "width": 4096, "pitch": 4096, "dtype": "bfloat16"},
        # decoding: one request's down projection, eight requests' merged gate and up projection, 64 requests' output projection
        {"name": "product_1x4096x12288", "kind": "product", "rows": 1, "features": 4096, "width": 12288, "out": "bfloat16"},
        {"name": "product_8x24576x4096", "kind": "product", "rows": 8, "features": 24576, "width": 4096, "out": "bfloat16"},
        {"name": "product_64x4096x4096", "kind": "product", "rows": 64, "features": 4096, "width": 4096, "out": "bfloat16"},
        # nothing is a multiple of anything, float32 results
        {"name": "product_300x1111x2008_f32", "kind": "product", "rows": 300, "features": 1111, "width": 2008, "out": "float32"},
        # a prompt portion of 2,048 tokens, and a step of four of them at the widest sizes
        {"name": "product_2048x24576x4096", "kind": "product", "rows": 2048, "features": 24576, "width": 4096, "out": "bfloat16"},
        {"name": "product_8192x5120x25600", "kind": "product", "rows": 8192, "features": 5120, "width": 25600, "out": "bfloat16"},
        # the feed-forward of a layer: one token, a small batch, a prompt portion
        {"name": "feed_forward_1x4096x12288", "kind": "feed_forward", "rows": 1, "width": 4096, "inner": 12288},
        {"name": "feed_forward_24x1024x2824", "kind": "feed_forward", "rows": 24, "width": 1024, "inner": 2824},
        {"name": "feed_forward_2048x4096x12288", "kind": "feed_forward", "rows": 2048, "width": 4096, "inner": 12288},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["quantise", "product", "product", "feed_forward"])
    if kind == "quantise":
        width = _log_uniform(rng, 40, 25600)
        rows = _log_uniform(rng, 1, min(32768, 24576 * 4096 // width))
        return {"kind": kind, "rows": rows, "width": width, "pitch": width + rng.choice([0, 0, 8, 333]),
                "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}
    if kind == "product":
        rows, width = _log_uniform(rng, 1, 8192), _log_uniform(rng, 64, 25600)
        if rng.random() < 0.5:
            width = max(64, width // 64 * 64)
        features = _log_uniform(rng, 64, min(25600, 8192 * 5120 * 25600 // (rows * width)))
        return {"kind": kind, "rows": rows, "features": features, "width": width,
                "out": rng.choice(["bfloat16", "bfloat16", "float32"])}
    rows, width = _log_uniform(rng, 1, 4096), 8 * _log_uniform(rng, 16, 640)
    return {"kind": kind, "rows": rows, "width": width, "inner": 8 * _log_uniform(rng, 16, 1600)}


def work(case):
    held = 0.5 + 1.0 / BLOCK  # bytes that a value takes in this form
    t, k = case["rows"], case["width"]
    if case["kind"] == "quantise":
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": t * k * (size + held + 2), "flops": 4 * t * k}
    if case["kind"] == "product":
        n = case["features"]
        return {"bytes": (t + n) * k * held + t * n * (2 if case["out"] == "bfloat16" else 4), "flops": 2 * t * n * k}
    i = case["inner"]
    return {"bytes": 3 * i * k * held + t * k * (4 + 4 + 2 + 2) + 4 * k, "flops": 6 * t * i * k}


# ---------------------------------------------------------------------- the plain form
def _scale_of(byte):
    """2^(byte - 127) as float32, 255: NaN."""
    b = byte.to(torch.int32)
    power = (b << 23).view(torch.float32)
    return torch.where(b == 0, 2.0 ** -127, torch.where(b == 255, math.nan, power))


def _round_rows(x):
    """The codes [R, 32 B] and the scales' bytes [R, B] of float32 rows [R, K]."""
    r, k = x.shape
    blocks = -(-k // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - k)).view(r, blocks, BLOCK)
    top = x.abs().amax(-1).view(torch.int32)  # for floats that are not negative the bits are in the numbers' order
    byte = torch.where(top >= 0x7F800000, 255, (((top + 0x1FFFFF) >> 23) - 2).clamp(min=0))
    a = (x / _scale_of(byte)[..., None]).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = code + 8 * (torch.signbit(x) & (byte != 255)[..., None]).to(torch.uint8)
    return code.view(r, blocks * BLOCK), byte.to(torch.uint8)


def _lay_out(code, byte):
    """Codes and scales as they are held."""
    r, blocks = byte.shape
    codes = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()
    tiles, across = -(-r // TILE_ROWS), -(-blocks // TILE_BLOCKS)
    full = torch.nn.functional.pad(byte, (0, across * TILE_BLOCKS - blocks, 0, tiles * TILE_ROWS - r))
    scales = full.view(tiles, 4, 32, across, 4).permute(0, 3, 2, 1, 4).reshape(tiles, across, 512).contiguous()
    return codes, scales


def _values(codes, scales, width, grid):
    """What the held rows stand for, float32 [R, width]."""
    r, blocks = codes.shape[0], -(-width // BLOCK)
    tiles, across = scales.shape[:2]
    byte = scales.view(tiles, across, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles * TILE_ROWS, across * TILE_BLOCKS)
    code = torch.stack([codes & 15, codes >> 4], dim=-1).view(r, blocks, BLOCK)
    v = grid[code.int()] * _scale_of(byte[:r, :blocks])[..., None]
    return v.view(r, blocks * BLOCK)[:, :width]


def _plain(s):
    c = s["case"]
    if c["kind"] == "quantise":
        x = s["x"].float()
        code, byte = _round_rows(x)
        v = s["grid"][code.int()].view(*byte.shape, BLOCK) * _scale_of(byte)[..., None]
        return {"values": v.view(x.shape[0], -1)[:, :c["width"]].to(torch.bfloat16)}
    if c["kind"] == "product":
        x = _values(s["x_codes"], s["x_scales"], c["width"], s["grid"])
        w = _values(s["w_codes"], s["w_scales"], c["width"], s["grid"])
        return {"y": (x @ w.t()).to(DT[c["out"]])}
    stream = s["stream"] + s["delta"].float()
    h = stream / torch.sqrt(stream.square().mean(-1, keepdim=True) + EPS) * s["norm"]
    h = _values(*_lay_out(*_round_rows(h)), c["width"], s["grid"])
    both = h @ _values(s["gate_up_codes"], s["gate_up_scales"], c["width"], s["grid"]).t()
    both = both.view(c["rows"], c["inner"] // 8, 2, 8)
    gate, up = both[:, :, 0].reshape(c["rows"], -1), both[:, :, 1].reshape(c["rows"], -1)
    a = gate / (1.0 + torch.exp(-gate)) * up
    a = _values(*_lay_out(*_round_rows(a)), c["inner"], s["grid"])
    y = a @ _values(s["down_codes"], s["down_scales"], c["inner"], s["grid"]).t()
    return {"stream": stream, "y": y.to(torch.bfloat16)}


# ---------------------------------------------------------------------- a user's state and calls
def _random(rows, width, g, spread=1.0):
    """Activations: normal, with a width of their own in each feature, a few of them many times the others'."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    return x * torch.exp(0.7 * torch.randn(width, generator=g, device="cuda")) * spread


def _weight(rows, width, g):
    """A weight in the form that it is held in (rounded in pieces, so that the float32 copy stays small)."""
    codes, bytes_ = [], []
    for at in range(0, rows, 4096):
        code, byte = _round_rows(torch.randn(min(4096, rows - at), width, generator=g, device="cuda") * width ** -0.5)
        codes.append(code)
        bytes_.append(byte)
    return _lay_out(torch.cat(codes), torch.cat(bytes_))


def _empty_rows(rows, width):
    tiles, across = -(-rows // TILE_ROWS), -(-width // (BLOCK * TILE_BLOCKS))
    return (torch.zeros(rows, -(-width // BLOCK) * 16, dtype=torch.uint8, device="cuda"),
            torch.zeros(tiles, across, 512, dtype=torch.uint8, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, k = case["rows"], case["width"]
    s = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device="cuda"),
         "grid": torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")}
    if case["kind"] == "quantise":
        s["x"] = _random(t, case["pitch"], g).to(DT[case["dtype"]])[:, :k]
        s["codes"], s["scales"] = _empty_rows(t, k)
        s["values"] = torch.empty(t, k, dtype=torch.bfloat16, device="cuda")
    elif case["kind"] == "product":
        s["x_codes"], s["x_scales"] = _lay_out(*_round_rows(_random(t, k, g)))
        s["w_codes"], s["w_scales"] = _weight(case["features"], k, g)
        s["y"] = torch.empty(t, case["features"], dtype=DT[case["out"]], device="cuda")
    else:
        i = case["inner"]
        s["stream"] = _random(t, k, g, 2.0)
        s["delta"] = _random(t, k, g, 0.3).to(torch.bfloat16)
        s["norm"] = 1.0 + 0.1 * torch.randn(k, generator=g, device="cuda")
        s["gate_up_codes"], s["gate_up_scales"] = _weight(2 * i, k, g)
        s["down_codes"], s["down_scales"] = _weight(k, i, g)
        s["stream_out"] = torch.empty_like(s["stream"])
        s["h_codes"], s["h_scales"] = _empty_rows(t, k)
        s["a_codes"], s["a_scales"] = _empty_rows(t, i)
        s["y"] = torch.empty(t, k, dtype=torch.bfloat16, device="cuda")
    return s


def _own(s):
    from qwen3_from_scratch_b200.kernels import ops
    c = s["case"]
    if c["kind"] == "quantise":
        ops.fp4_quantise(s["x"], ops.Fp4Rows(s["codes"], s["scales"], c["width"]), values=s["values"])
        return {"values": s["values"]}
    if c["kind"] == "product":
        ops.fp4_product(ops.Fp4Rows(s["x_codes"], s["x_scales"], c["width"]),
                        ops.Fp4Rows(s["w_codes"], s["w_scales"], c["width"]), s["y"], s["status"])
        return {"y": s["y"]}
    ops.fp4_feed_forward(s["stream"], s["delta"], s["norm"], EPS,
                         ops.Fp4Rows(s["gate_up_codes"], s["gate_up_scales"], c["width"]),
                         ops.Fp4Rows(s["down_codes"], s["down_scales"], c["inner"]),
                         ops.Fp4Rows(s["h_codes"], s["h_scales"], c["width"]),
                         ops.Fp4Rows(s["a_codes"], s["a_scales"], c["inner"]),
                         s["y"], s["status"], activation="silu", stream_out=s["stream_out"])
    return {"stream": s["stream_out"], "y": s["y"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------- the definition in 64 bits
def _stood_for(x):
    """What float64 rows [R, K] are rounded to, float64, by comparing every value with the eight of the format."""
    r, k = x.shape
    out = torch.zeros_like(x)
    whole = torch.zeros(r, -(-k // 32) * 32, dtype=torch.float64, device=x.device)
    whole[:, :k] = x
    b = whole.view(r, -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    # the smallest n with top <= 7 2^n, by frexp: top / 7 = f 2^e with 1/2 <= f < 1, and a power of two itself at f = 1/2
    f, e = torch.frexp(top / 7.0)
    n = torch.where(f == 0.5, e - 1, e).clamp(min=-127)
    n = torch.where(top == 0, torch.full_like(n, -127), n)
    unit = torch.ldexp(torch.ones_like(top), n)
    q = (b / unit).abs()
    held = torch.zeros_like(q)
    steps = ((0.25, False, 0.5), (0.75, True, 1.0), (1.25, False, 1.5), (1.75, True, 2.0), (2.5, False, 3.0),
             (3.5, True, 4.0), (5.0, False, 6.0))  # from where on, itself included, what
    for limit, with_it, value in steps:
        held = torch.where((q >= limit) if with_it else (q > limit), torch.full_like(q, value), held)
    out.copy_((torch.sign(b) * held * unit).view(r, -1)[:, :k])
    return out


def _read(codes, scales, k):
    """Held rows as float64, bit by bit."""
    r, dev = codes.shape[0], codes.device
    col, row = torch.arange(k, device=dev), torch.arange(r, device=dev)
    nibble = (codes[:, col // 2].int() >> (4 * (col % 2))[None, :].int()) & 15
    exponent, half = (nibble >> 1) & 3, nibble & 1
    size = torch.where(exponent == 0, 0.5 * half.double(), (1.0 + 0.5 * half.double()) * 2.0 ** (exponent - 1).double())
    sign = 1.0 - 2.0 * (nibble >> 3).double()
    j = torch.arange(-(-k // 32), device=dev)
    flat = scales.reshape(-1)
    at = ((row[:, None] // 128 * scales.shape[1] + j[None, :] // 4) * 512 + 16 * (row[:, None] % 32)
          + 4 * (row[:, None] % 128 // 32) + j[None, :] % 4)
    unit = torch.ldexp(torch.ones(r, len(j), dtype=torch.float64, device=dev), flat[at].int() - 127)
    return sign * size * unit.repeat_interleave(32, dim=1)[:, :k]


def _times(x, codes, scales, k):
    """x w^T in 64 bits, some rows of the weight at a time."""
    return torch.cat([x @ _read(codes[at:at + 2048], scales[at // 128:(at + 2048) // 128], k).t()
                      for at in range(0, codes.shape[0], 2048)], dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    k = case["width"]
    if case["kind"] == "quantise":
        return {"values": torch.cat([_stood_for(x.double()) for x in s["x"].split(2048)])}
    if case["kind"] == "product":
        return {"y": _times(_read(s["x_codes"], s["x_scales"], k), s["w_codes"], s["w_scales"], k)}
    stream = s["stream"].double() + s["delta"].double()
    h = stream * (stream.pow(2).sum(1, keepdim=True) / k + EPS).rsqrt() * s["norm"].double()
    both = _times(_stood_for(h), s["gate_up_codes"], s["gate_up_scales"], k).view(case["rows"], -1, 16)
    a = (torch.sigmoid(both[..., :8]) * both[..., :8] * both[..., 8:]).reshape(case["rows"], -1)
    return {"stream": stream, "y": _times(_stood_for(a), s["down_codes"], s["down_scales"], case["inner"])}
