"""Rows in microscaled 4-bit floating point and the products of such rows, against the definition in 64 bits."""

import math

import pytest
import torch

import plain_fp4 as plain

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def ops():
    from qwen3_from_scratch_b200.kernels import ops as o
    return o


def status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def normal(rows, width, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g)
    return x * torch.exp(0.7 * torch.randn(width, generator=g)) if spread else x


def held(x):
    """The rows of a CPU tensor, rounded on the GPU, and what they stand for in float64."""
    o = ops()
    r = o.fp4_rows(x.shape[0], x.shape[1], "cuda")
    o.fp4_quantise(x.cuda(), r)
    return r, plain.read(r.codes, r.scales, x.shape[1])[0]


def junk_rows(rows, width):
    """Memory for rows with every byte set: what a kernel does not write stays visible."""
    r = ops().fp4_rows(rows, width, "cuda")
    r.codes.fill_(0xA5)
    r.scales.fill_(0xFF)
    return r


def pad_is_zero(r):
    """Codes beyond the width and the scales of blocks beyond it."""
    rows, k = r.codes.shape[0], r.width
    nibbles = torch.stack([r.codes & 15, r.codes >> 4], dim=-1).reshape(rows, -1).cpu()
    across = r.scales.shape[1]
    _, byte = plain.read(torch.zeros(rows, across * 64, dtype=torch.uint8), r.scales, across * 128)
    return bool((nibbles[:, k:] == 0).all()) and bool((byte[:, -(-k // 32):] == 0).all())


# ---------------------------------------------------------------- rounding
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 31), (1, 32), (3, 33), (2, 127), (5, 128), (4, 129), (2, 256), (130, 264),
                                        (129, 300), (7, 1000), (3, 4104), (257, 96), (1, 12288)])
def test_quantise(dtype, rows, width):
    x = normal(rows, width, rows * 10007 + width).to(DT[dtype])
    r = junk_rows(rows, width)
    values = torch.empty(rows, width, dtype=torch.float32, device="cuda")
    ops().fp4_quantise(x.cuda(), r, values=values)
    want = plain.rounded(x.double())
    got, _ = plain.read(r.codes, r.scales, width)
    assert torch.equal(got, want)  # rounding is exact: no tolerance
    assert torch.equal(values.cpu().double(), want)
    assert pad_is_zero(r)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("pitch,start", [(300, 0), (301, 0), (304, 8), (333, 1), (320, 3)])
def test_quantise_columns_of_a_wider_buffer(dtype, pitch, start):
    wide = normal(9, pitch, pitch).to(DT[dtype])
    width = 290
    x = wide.cuda()[:, start:start + width]
    r = junk_rows(9, width)
    values = torch.empty(9, width, dtype=torch.bfloat16, device="cuda")
    ops().fp4_quantise(x, r, values=values)
    want = plain.rounded(wide[:, start:start + width].double())
    assert torch.equal(plain.read(r.codes, r.scales, width)[0], want)
    assert torch.equal(values.cpu().double(), want)


def test_quantise_ties_ends_and_signs():
    """Every boundary between two codes at several scales, the values around the boundary between two scales, zeros of both
    signs, the smallest and the largest floats."""
    rows = []
    for e in (-126, -100, -3, 0, 40, 120):
        unit = 2.0 ** e
        row = [s * m * unit for m in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5) for s in (1, -1)]
        rows.append(row + [7.0 * unit] + [0.0] * (32 - len(row) - 1))
        rows.append(row + [math.nextafter(7.0, 8.0) * unit * (1 + 2.0 ** -22)] + [-0.0] * (32 - len(row) - 1))
    rows += [[0.0] * 32, [-0.0] * 32, [2.0 ** -149] * 32, [2.0 ** -127, -(2.0 ** -128)] * 16, [2.0 ** -126 * 1.75] * 32]
    x = torch.tensor(rows, dtype=torch.float64).float()
    assert bool(torch.isfinite(x).all())
    r = junk_rows(x.shape[0], 32)
    ops().fp4_quantise(x.cuda(), r)
    got, byte = plain.read(r.codes, r.scales, 32)
    assert torch.equal(got, plain.rounded(x.double()))
    assert torch.equal(byte[:, 0].int() - 127, plain.scale_exponents(x.double())[:, 0])
    big = torch.full((1, 32), torch.finfo(torch.float32).max).cuda()
    b = junk_rows(1, 32)
    ops().fp4_quantise(big, b)  # the largest float has a scale of its own; its value rounds up to 4 x 2^126
    assert int(b.scales.reshape(-1)[0]) == 253 and bool((b.codes == 0x66).all())


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("width", [1, 7, 9, 255, 257, 263, 1023, 1025, 1031, 2049, 2300])
def test_quantise_values_off_every_boundary(width, out):
    """Values whose rows begin at every place within 16 bytes: those that the codes stand for, and nothing around them is touched."""
    x = normal(18, width, width)
    own = ops().fp4_rows(18, width, "cuda")
    ops().fp4_quantise(x.cuda(), own)
    want, _ = plain.read(own.codes, own.scales, width)
    for start in range(0, 9):
        room = torch.full((18 * width + 64,), 3.0, dtype=DT[out], device="cuda")
        values = room[start:start + 18 * width].view(18, width)
        ops().fp4_quantise(x.cuda(), ops().fp4_rows(18, width, "cuda"), values)
        assert torch.equal(values.cpu().double(), want), start
        assert bool((room[:start] == 3).all()) and bool((room[start + 18 * width:] == 3).all()), start


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("dtype", list(DT))
def test_quantise_values_of_the_largest_numbers(dtype, out):
    """In a block that reaches beyond 1.75 x 2^127 values from there on are rounded to 4 x 2^126, which is no float: infinity with its
    sign.  Everything else is exact."""
    top = 2.0 ** 127
    x = torch.zeros(3, 64)
    x[0, :6] = torch.tensor([1.9921875, -1.9921875, 1.75, 1.5, -1.0, 0.125]) * top
    x[1, :3] = torch.tensor([1.75, -1.75, 0.25]) * top  # 7 x 2^125
    x[2, 32:34] = torch.tensor([-1.9921875, 0.5]) * top
    x = x.to(DT[dtype])
    assert bool(torch.isfinite(x).all())
    r, values = junk_rows(3, 64), torch.empty(3, 64, dtype=DT[out], device="cuda")
    ops().fp4_quantise(x.cuda(), r, values=values)
    want = plain.rounded(x.double())
    assert torch.equal(plain.read(r.codes, r.scales, 64)[0], want)
    assert torch.equal(values.cpu().double(), want.float().double())
    assert int(torch.isinf(values).sum()) == 4 and bool(torch.isfinite(values[1]).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_quantise_what_is_not_finite(bad):
    x = normal(3, 100, 5)
    x[1, 40] = bad
    r = junk_rows(3, 100)
    values = torch.empty(3, 100, device="cuda")
    ops().fp4_quantise(x.cuda(), r, values=values)
    clean = x.clone()
    clean[1, 32:64] = 0
    want = plain.rounded(clean.double())
    want[1, 32:64] = math.nan
    assert torch.equal(values.cpu().double().nan_to_num(77.0), want.nan_to_num(77.0))
    assert torch.equal(plain.read(r.codes, r.scales, 100)[0].nan_to_num(77.0), want.nan_to_num(77.0))


# ---------------------------------------------------------------- the norm
@pytest.mark.parametrize("dtype", [None, "float32", "bfloat16"])
@pytest.mark.parametrize("rows,width", [(1, 8), (2, 33), (5, 1000), (130, 264), (3, 4096), (2, 5121), (2, 12288), (1, 32768)])
def test_add_rmsnorm(dtype, rows, width):
    stream = normal(rows, width, 3 * rows + width) * 2
    delta = None if dtype is None else (normal(rows, width, 7 * width) * 0.3).to(DT[dtype])
    w = 1 + 0.1 * normal(1, width, 11, spread=False)[0]
    total = stream if delta is None else stream + delta.float()
    s = total.double()
    h = s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-6) * w.double()
    # the sum of squares of positive terms, a root, a quotient and two products: under 20 roundings of 2^-24
    low, high = plain.between(h, h.abs() * 20 * 2.0 ** -24)
    d = None if delta is None else delta.cuda()
    other, r = torch.empty(rows, width, device="cuda"), junk_rows(rows, width)
    ops().fp4_add_rmsnorm(stream.cuda(), d, w.cuda(), r, 1e-6, stream_out=other)
    got, _ = plain.read(r.codes, r.scales, width)
    assert torch.equal(other.cpu(), total)
    assert bool(((got >= low) & (got <= high)).all())
    assert pad_is_zero(r)
    here, again = stream.cuda(), junk_rows(rows, width)
    ops().fp4_add_rmsnorm(here, d, w.cuda(), again, 1e-6)
    assert torch.equal(here, other) and torch.equal(again.codes, r.codes)


# ---------------------------------------------------------------- products
def product_tolerance(x, w):
    """Per result: products of held values are exact, a float32 sum of K of them is off by at most the number of its roundings
    times 2^-24 of the sum of their sizes; tensor cores add 64 at a time and may cut instead of round (2^-23)."""
    return (x.abs() @ w.abs().t()) * ((x.shape[1] + 63) // 64 + 8) * 2.0 ** -23


FORMS = [None, "few", "pair192", "pair256", "pair384"]
SIZES = [(1, 1, 1), (1, 8, 31), (1, 127, 32), (1, 130, 33), (2, 129, 64), (3, 64, 65), (7, 300, 127), (8, 128, 128), (9, 16, 129),
         (16, 256, 256), (17, 257, 257), (33, 200, 300), (64, 520, 1000), (65, 100, 2008), (128, 384, 512), (129, 129, 640),
         (200, 1111, 264), (300, 250, 4104), (512, 512, 1024), (700, 777, 776), (257, 1601, 160), (1030, 1400, 300)]


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("rows,features,width", SIZES)
def test_product(out, rows, features, width):
    """Every form at every size, whether or not it is the one that the size asks for."""
    x, xv = held(normal(rows, width, rows + width))
    w, wv = held(normal(features, width, features + 1, spread=False) * width ** -0.5)
    want, tol = xv @ wv.t(), product_tolerance(xv, wv)
    if out == "bfloat16":
        tol = tol + want.abs() * 2.0 ** -8
    for form in FORMS:
        if form == "pair384" and out == "float32":
            continue
        y = torch.full((rows, features), 7.0, dtype=DT[out], device="cuda")
        st = status()
        ops().fp4_product(x, w, y, st, form=form)
        assert int(st.item()) == 0
        assert bool(((y.cpu().double() - want).abs() <= tol).all()), form


@pytest.mark.parametrize("rows,features,width", [(128, 24600, 4096), (512, 28416, 4096), (768, 9440, 2056), (1025, 4736, 2048)])
def test_product_at_sizes_of_prompts(rows, features, width):
    """Where the rule takes pairs of CTAs with several tiles each; w repeats 300 rows in a random order, so that the definition in
    64 bits is a small product."""
    x, xv = held(normal(rows, width, 1))
    few = normal(300, width, 2, False) * width ** -0.5
    order = torch.randint(0, 300, (features,), generator=torch.Generator().manual_seed(3))
    w = ops().fp4_rows(features, width, "cuda")
    ops().fp4_quantise(few.cuda()[order.cuda()], w)
    wv = plain.rounded(few.double())
    want, tol = (xv @ wv.t()).cuda(), product_tolerance(xv, wv).cuda()
    want, tol = want[:, order.cuda()], tol[:, order.cuda()]
    for out in DT.values():
        y = torch.full((rows, features), 7.0, dtype=out, device="cuda")
        ops().fp4_product(x, w, y, status())
        bound = tol + want.abs() * 2.0 ** -8 if out == torch.bfloat16 else tol
        assert bool(((y.double() - want).abs() <= bound).all())


def test_products_of_more_rows_than_a_grid_of_small_tiles_has():
    """Over 65,535 tiles of 128 rows, narrow enough that small tiles would be the faster ones: the rows repeat 1,000 others, and hold
    whole numbers of up to 4, whose sums are exact in any order."""
    o, rows, width = ops(), 65535 * 128 + 1, 64
    g = torch.Generator().manual_seed(1)
    data, weight = (torch.randint(-4, 5, (n, width), generator=g).float() for n in (1000, 64))
    x, st = o.fp4_rows(rows, width, "cuda"), status()
    o.fp4_quantise(data.cuda()[torch.arange(rows, device="cuda") % 1000], x)
    w, some = held(weight)[0], held(data)[0]
    want, want4 = torch.empty(1000, 64, dtype=torch.bfloat16, device="cuda"), o.fp4_rows(1000, 32, "cuda")
    o.fp4_product(some, w, want, st)
    o.fp4_gated_product(some, w, want4, st)
    y, y4 = torch.empty(rows, 64, dtype=torch.bfloat16, device="cuda"), o.fp4_rows(rows, 32, "cuda")
    o.fp4_product(x, w, y, st)
    o.fp4_gated_product(x, w, y4, st)
    assert int(st.item()) == 0
    whole = rows // 1000 * 1000
    for got, of in ((y, want), (y4.codes, want4.codes)):
        assert bool((got[:whole].view(-1, 1000, got.shape[1]) == of).all()) and torch.equal(got[whole:], of[:rows - whole])
    with pytest.raises(o.KernelSizeError):
        o.fp4_product(x, w, y, st, form="few")


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("rows,features", [(1, 290), (40, 290), (300, 290), (300, 800)])
@pytest.mark.parametrize("start,more", [(0, 30), (8, 46), (3, 11)])
def test_product_into_columns(out, rows, features, start, more):
    x, xv = held(normal(rows, 200, rows))
    w, wv = held(normal(features, 200, 2, spread=False))
    end = start + features
    want = xv @ wv.t()
    tol = product_tolerance(xv, wv) + (want.abs() * 2.0 ** -8 if out == "bfloat16" else 0)
    for form in FORMS:
        if form == "pair384" and out == "float32":
            continue
        wide = torch.full((rows, features + more), 3.0, dtype=DT[out], device="cuda")
        ops().fp4_product(x, w, wide[:, start:end], status(), form=form)
        assert bool(((wide[:, start:end].cpu().double() - want).abs() <= tol).all()), form
        assert bool((wide[:, :start] == 3).all()) and bool((wide[:, end:] == 3).all()), form


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("rows", [1, 70, 300])
@pytest.mark.parametrize("features", [1, 15, 33, 191, 193, 257, 385, 450, 513])
def test_product_off_every_boundary(rows, features, out):
    """Rows that begin at every place within 32 bytes, in rows further apart than they are long: the same bits as in rows of their own,
    and nothing of what lies around them is touched."""
    x, _ = held(normal(rows, 96, rows))
    w, _ = held(normal(features, 96, 2, spread=False))
    for form in ("few", "pair192", "pair256", "pair384"):
        if form == "pair384" and out == "float32":
            continue
        own = torch.empty(rows, (features + 15) // 16 * 16, dtype=DT[out], device="cuda")
        ops().fp4_product(x, w, own[:, :features], status(), form=form)
        for start in range(0, 17):
            pitch = features + start + (5 * start + 3) % 17
            wide = torch.full((rows + 2, pitch), 3.0, dtype=DT[out], device="cuda")
            ops().fp4_product(x, w, wide[1:-1, start:start + features], status(), form=form)
            assert torch.equal(wide[1:-1, start:start + features], own[:, :features]), (form, start)
            wide[1:-1, start:start + features] = 3.0
            assert bool((wide == 3).all()), (form, start)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,features", [(5, 200), (300, 700)])
def test_product_rows_beyond_the_first(rows, features, form):
    """The first rows of a larger buffer whose other rows hold anything, their scales NaN."""
    width = 520
    whole = junk_rows(rows + 150, width)
    x = whole.first(rows)
    data = normal(rows, width, 4)
    ops().fp4_quantise(data.cuda(), x)
    w, wv = held(normal(features, width, 8))
    y = torch.empty(rows, features, device="cuda", dtype=torch.bfloat16)
    ops().fp4_product(x, w, y, status(), form=form)
    xv = plain.rounded(data.double())
    want = xv @ wv.t()
    assert bool(((y.cpu().double() - want).abs() <= product_tolerance(xv, wv) + want.abs() * 2.0 ** -8).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,features", [(3, 260), (300, 500)])
def test_product_of_what_is_not_finite(rows, features, form):
    """A NaN scale reaches the results of its row of x or of w, and no others."""
    xd, wd = normal(rows, 300, 1), normal(features, 300, 2)
    xd[1, 77], wd[130, 299] = math.inf, math.nan
    x, w = held(xd)[0], held(wd)[0]
    y = torch.empty(rows, features, device="cuda", dtype=torch.bfloat16)
    ops().fp4_product(x, w, y, status(), form=form)
    want = torch.zeros(rows, features, dtype=torch.bool)
    want[1], want[:, 130] = True, True
    assert torch.equal(torch.isnan(y).cpu(), want)
    assert bool(torch.isfinite(y.cpu()[~want]).all())


def interleaved(gate, up):
    i = gate.shape[0]
    return torch.cat([gate.view(i // 8, 8, -1), up.view(i // 8, 8, -1)], dim=1).reshape(2 * i, -1)


def gated_bounds(xv, wv, act):
    """act(gate) * up in float64 and how far the kernel's may be from it: the products' own errors carried through (none of the
    gates is steeper than 1.13), and 16 roundings of 2^-24 and the fast exponential's 2^-21 in the gate itself."""
    both, tol = xv @ wv.t(), product_tolerance(xv, wv)
    split = [t.view(t.shape[0], -1, 2, 8) for t in (both, tol)]
    gate, up, dg, du = (t[:, :, k].reshape(t.shape[0], -1) for t in split for k in (0, 1))
    if act == "silu":
        f = gate * torch.sigmoid(gate)
    elif act == "relu":
        f = gate.clamp(min=0)
    else:
        f = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
    a = f * up
    # the gelu's 1 + tanh(y) loses what is below 2^-24 of 1, times the gate
    lost = gate.abs() * up.abs() * 2.0 ** -22 if act == "gelu_tanh" else 0
    return a, 1.13 * dg * (up.abs() + du) + f.abs() * du + a.abs() * 2.0 ** -19 + lost


@pytest.mark.parametrize("act", ["silu", "relu", "gelu_tanh"])
@pytest.mark.parametrize("rows,inner,width", [(1, 8, 32), (1, 64, 100), (3, 40, 264), (8, 136, 1024), (24, 200, 520), (33, 504, 256),
                                              (130, 1000, 384), (300, 320, 600), (513, 600, 512), (300, 1504, 136), (1040, 1736, 1300)])
def test_gated_product(act, rows, inner, width):
    x, xv = held(normal(rows, width, rows))
    w, wv = held(interleaved(normal(inner, width, 1, False), normal(inner, width, 2, False)) * width ** -0.5)
    a, slack = gated_bounds(xv, wv, act)
    low, high = plain.between(a, slack)
    for form in (None, "few", "pair192", "pair256"):
        r = junk_rows(rows, inner)
        st = status()
        ops().fp4_gated_product(x, w, r, st, activation=act, form=form)
        got, _ = plain.read(r.codes, r.scales, inner)
        assert int(st.item()) == 0
        assert bool(((got >= low) & (got <= high)).all()), form
        assert pad_is_zero(r), form


@pytest.mark.parametrize("rows", [24, 25, 32, 33, 63, 64, 65, 96, 127, 128, 129, 152, 200])
@pytest.mark.parametrize("inner,width", [(8, 40), (24, 256), (72, 200), (104, 256), (136, 64), (4104, 1024)])
def test_gated_product_of_a_few_tiles_of_rows(rows, inner, width):
    """Rows that are finished by sixteen lanes and rows that a lane finishes alone, on both sides of every count where the one takes
    over from the other or the next warp's rows begin, with last blocks that are not full."""
    x, xv = held(normal(rows, width, rows))
    w, wv = held(interleaved(normal(inner, width, 1, False), normal(inner, width, 2, False)) * width ** -0.5)
    a, slack = gated_bounds(xv, wv, "silu")
    low, high = plain.between(a, slack)
    r, st = junk_rows(rows, inner), status()
    ops().fp4_gated_product(x, w, r, st, form="few")
    got, _ = plain.read(r.codes, r.scales, inner)
    assert int(st.item()) == 0
    assert bool(((got >= low) & (got <= high)).all())
    assert pad_is_zero(r)


@pytest.mark.parametrize("rows", [20, 60, 130])
def test_gated_product_of_a_few_tiles_of_what_is_not_finite(rows):
    w, _ = held(normal(64, 64, 3, False))
    values = normal(rows, 64, rows)
    values[1, 5] = math.nan
    x, _ = held(values)
    r, st = junk_rows(rows, 32), status()
    ops().fp4_gated_product(x, w, r, st, form="few")
    assert int(st.item()) == 0
    got, byte = plain.read(r.codes, r.scales, 32)
    assert bool(torch.isnan(got[1]).all())
    assert bool(torch.isfinite(got[torch.arange(rows, device=got.device) != 1]).all())


@pytest.mark.parametrize("form", [None, "pair192", "pair256"])
@pytest.mark.parametrize("rows", [2, 260])
def test_gated_product_of_what_is_not_finite(rows, form):
    xd = normal(rows, 128, 1)
    xd[1, 5] = math.nan
    x = held(xd)[0]
    w = held(interleaved(normal(72, 128, 1, False), normal(72, 128, 2, False)))[0]
    r = junk_rows(rows, 72)
    ops().fp4_gated_product(x, w, r, status(), form=form)
    got, byte = plain.read(r.codes, r.scales, 72)
    assert bool((byte[1] == 255).all())
    assert bool(torch.isfinite(got[0]).all()) and bool((byte[0] < 255).all())


@pytest.mark.parametrize("act", ["silu", "relu", "gelu_tanh"])
@pytest.mark.parametrize("half", ["gate", "up"])
@pytest.mark.parametrize("rows,form", [(3, "few"), (3, None), (40, "few"), (260, "few"), (260, "pair192"), (260, "pair256")])
def test_gated_product_of_one_row_that_is_not_finite(rows, form, half, act):
    """A NaN in one gate or up row alone: the block of results that holds its column is NaN in every row, no other is."""
    parts = {"gate": normal(72, 2304, 1, False), "up": normal(72, 2304, 2, False)}
    parts[half][37, 9] = math.nan
    x, w = held(normal(rows, 2304, 3))[0], held(interleaved(parts["gate"], parts["up"]))[0]
    r, st = junk_rows(rows, 72), status()
    ops().fp4_gated_product(x, w, r, st, activation=act, form=form)
    got, byte = plain.read(r.codes, r.scales, 72)
    assert int(st.item()) == 0
    assert bool((byte[:, 1] == 255).all()) and bool((byte[:, [0, 2]] < 255).all())
    assert bool(torch.isnan(got[:, 32:64]).all()) and bool(torch.isfinite(got[:, :32]).all())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,width,inner", [(1, 8, 8), (1, 256, 520), (1, 4096, 1200), (3, 4104, 200), (7, 8192 // 2, 328), (24, 512, 1000), (24, 1000, 504),
                                              (32, 1024, 72), (33, 1024, 72), (4, 8192, 160), (9, 4096, 160), (2, 12288, 64), (2, 100, 80),
                                              (300, 264, 328)])
def test_feed_forward_is_its_parts(dtype, rows, width, inner):
    o = ops()
    stream, delta = normal(rows, width, 1).cuda(), (normal(rows, width, 2) * 0.3).to(DT[dtype]).cuda()
    norm = (1 + 0.1 * normal(1, width, 3, False)[0]).cuda()
    gu = held(interleaved(normal(inner, width, 4, False), normal(inner, width, 5, False)) * width ** -0.5)[0]
    down = held(normal(width, inner, 6, False) * inner ** -0.5)[0]
    h, a = o.fp4_rows(rows, width, "cuda"), o.fp4_rows(rows, inner, "cuda")
    y, s, st = torch.empty(rows, width, dtype=DT[dtype], device="cuda"), torch.empty_like(stream), status()
    o.fp4_feed_forward(stream, delta, norm, 1e-6, gu, down, h, a, y, st, stream_out=s)
    h2, a2, y2, s2 = o.fp4_rows(rows, width, "cuda"), o.fp4_rows(rows, inner, "cuda"), torch.empty_like(y), torch.empty_like(stream)
    o.fp4_add_rmsnorm(stream, delta, norm, h2, 1e-6, stream_out=s2)
    o.fp4_gated_product(h2, gu, a2, st)
    o.fp4_product(a2, down, y2, st)
    assert int(st.item()) == 0
    assert torch.equal(s, s2) and torch.equal(h.codes, h2.codes) and torch.equal(a.codes, a2.codes) and torch.equal(y, y2)
    for one, other in ((h, h2), (a, a2)):
        assert torch.equal(plain.read(one.codes, one.scales, one.width)[1], plain.read(other.codes, other.scales, other.width)[1])
    # and against 64 bits: as the last product of what the gate left
    want = plain.read(a.codes, a.scales, inner)[0] @ plain.read(down.codes, down.scales, inner)[0].t()
    tol = product_tolerance(plain.read(a.codes, a.scales, inner)[0], plain.read(down.codes, down.scales, inner)[0])
    assert bool(((y.cpu().double() - want).abs() <= tol + (want.abs() * 2.0 ** -8 if dtype == "bfloat16" else 0)).all())
    junk = [junk_rows(rows, width), junk_rows(rows, inner)]
    y.fill_(3)
    o.fp4_feed_forward(stream.clone(), delta.clone(), norm, 1e-6, gu, down, *junk, delta, st, stream_out=s)  # the output over delta
    assert torch.equal(delta, y2) and torch.equal(s, s2) and pad_is_zero(junk[0]) and pad_is_zero(junk[1])
    o.fp4_feed_forward(s, None, norm, 1e-6, gu, down, h, a, y, st, stream_out=stream)  # no delta
    assert torch.equal(stream, s2) and torch.equal(y, y2)


@pytest.mark.parametrize("rows,width", [(1, 256), (24, 512), (40, 512)])
def test_feed_forward_updates_the_stream_in_place(rows, width):
    o, inner = ops(), 264
    stream, delta = normal(rows, width, 1).cuda(), (normal(rows, width, 2) * 0.3).cuda()
    total = stream + delta
    norm = torch.ones(width, device="cuda")
    gu = held(interleaved(normal(inner, width, 4, False), normal(inner, width, 5, False)) * width ** -0.5)[0]
    down = held(normal(width, inner, 6, False) * inner ** -0.5)[0]
    h, a, st = o.fp4_rows(rows, width, "cuda"), o.fp4_rows(rows, inner, "cuda"), status()
    want, y = torch.empty_like(delta), torch.empty_like(delta)
    o.fp4_feed_forward(total.clone(), None, norm, 1e-6, gu, down, h, a, want, st)
    o.fp4_feed_forward(stream, delta, norm, 1e-6, gu, down, h, a, y, st)
    assert torch.equal(stream, total) and torch.equal(y, want) and int(st.item()) == 0


@pytest.mark.parametrize("rows", [1, 20])
def test_feed_forward_right_behind_what_rounds_its_weights(rows):
    o, width, inner = ops(), 1024, 2000
    stream, norm = normal(rows, width, 1).cuda(), torch.ones(width, device="cuda")
    wide = interleaved(normal(inner, width, 4, False), normal(inner, width, 5, False)).cuda()
    narrow = normal(width, inner, 6, False).cuda()
    gu, down = o.fp4_rows(2 * inner, width, "cuda"), o.fp4_rows(width, inner, "cuda")
    h, a, st = o.fp4_rows(rows, width, "cuda"), o.fp4_rows(rows, inner, "cuda"), status()
    want = y = None
    for _ in range(4):
        gu.codes.fill_(0xA5)
        down.codes.fill_(0xA5)
        y = torch.empty(rows, width, device="cuda")
        torch.cuda.synchronize()
        o.fp4_quantise(narrow, down)
        o.fp4_quantise(wide, gu)
        if want is None:
            torch.cuda.synchronize()
        o.fp4_feed_forward(stream, None, norm, 1e-6, gu, down, h, a, y, st)
        want = y if want is None else want
        assert torch.equal(y, want)


def test_feed_forward_gives_up_cleanly():
    o, rows, width, inner = ops(), 2, 2048, 520
    stream, norm = normal(rows, width, 1).cuda(), torch.ones(width, device="cuda")
    gu = held(interleaved(normal(inner, width, 4, False), normal(inner, width, 5, False)))[0]
    down = held(normal(width, inner, 6, False))[0]
    h, a, st = o.fp4_rows(rows, width, "cuda"), o.fp4_rows(rows, inner, "cuda"), status()
    want, y = (torch.empty(rows, width, device="cuda") for _ in range(2))
    o.fp4_feed_forward(stream, None, norm, 1e-6, gu, down, h, a, want, st)
    try:
        o.set_wait_test(limit=1 << 14, drop_copy=0)  # a block may have one stage only
        o.fp4_feed_forward(stream, None, norm, 1e-6, gu, down, h, a, y, st)
        torch.cuda.synchronize()
        word = int(st.item())
    finally:
        o.set_wait_test()
    assert word & 16, f"status {word}: the time-out bit is not set"
    st.zero_()
    o.fp4_feed_forward(stream, None, norm, 1e-6, gu, down, h, a, y, st)
    assert torch.equal(y, want) and int(st.item()) == 0


# ---------------------------------------------------------------- calls
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,features", [(4, 600), (333, 1600)])
def test_the_same_inputs_give_the_same_bits_on_any_stream(rows, features, form):
    x, w = held(normal(rows, 2000, 1))[0], held(normal(features, 2000, 2))[0]
    first = torch.empty(rows, features, device="cuda", dtype=torch.bfloat16)
    ops().fp4_product(x, w, first, status(), form=form)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    again = [torch.empty_like(first) for _ in range(4)]
    with torch.cuda.stream(side):
        for y in again:
            ops().fp4_product(x, w, y, status(), form=form)
    side.synchronize()
    assert all(torch.equal(first, y) for y in again)


@pytest.mark.parametrize("rows", [3, 300])
def test_a_product_right_behind_what_rounds_its_w(rows):
    """The product reads w ahead of the kernel before it only where that kernel did not write it."""
    o = ops()
    x, xv = held(normal(rows, 4096, 1))
    data = normal(5000, 4096, 2, False).cuda()
    w, y, st = junk_rows(5000, 4096), torch.empty(rows, 5000, device="cuda"), status()
    want = torch.empty_like(y)
    o.fp4_quantise(data, w)
    torch.cuda.synchronize()
    o.fp4_product(x, w, want, st)
    for _ in range(5):
        w.codes.fill_(0xA5)
        o.fp4_quantise(data, w)
        o.fp4_product(x, w, y, st)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_no_rows_is_no_work():
    o = ops()
    empty, st = o.fp4_rows(0, 64, "cuda"), status()
    o.fp4_quantise(torch.empty(0, 64, device="cuda"), empty)
    o.fp4_product(empty, o.fp4_rows(32, 64, "cuda"), torch.empty(0, 32, device="cuda"), st)
    o.fp4_gated_product(empty, o.fp4_rows(32, 64, "cuda"), o.fp4_rows(0, 16, "cuda"), st)
    o.fp4_add_rmsnorm(torch.empty(0, 64, device="cuda"), None, torch.ones(64, device="cuda"), empty, 1e-6)


def test_refusals():
    o = ops()
    x, w, y, st = o.fp4_rows(4, 64, "cuda"), o.fp4_rows(32, 64, "cuda"), torch.empty(4, 32, device="cuda"), status()
    with pytest.raises(o.KernelError, match="expected"):
        o.fp4_product(x, o.fp4_rows(32, 96, "cuda"), y, st)
    with pytest.raises(o.KernelError, match="out"):
        o.fp4_product(x, w, torch.empty(4, 31, device="cuda"), st)
    with pytest.raises(o.KernelError, match="out"):
        o.fp4_product(x, w, torch.empty(32, 4, device="cuda").t(), st)
    with pytest.raises(o.KernelError, match="float32 or bfloat16"):
        o.fp4_product(x, w, y.half(), st)
    with pytest.raises(o.KernelError, match="codes"):
        o.fp4_product(o.Fp4Rows(x.codes[:, :16].contiguous(), x.scales, 64), w, y, st)
    with pytest.raises(o.KernelError, match="scales"):
        o.fp4_product(x, o.Fp4Rows(torch.zeros(200, 32, dtype=torch.uint8, device="cuda"), w.scales, 64),
                      torch.empty(4, 200, device="cuda"), st)
    with pytest.raises(o.KernelError, match="contiguous"):
        o.fp4_product(o.Fp4Rows(torch.zeros(4, 64, dtype=torch.uint8, device="cuda")[:, :32], x.scales, 64), w, y, st)
    odd = torch.zeros(4 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(4, 32)
    with pytest.raises(o.KernelError, match="misaligned"):
        o.fp4_product(o.Fp4Rows(odd, x.scales, 64), w, y, st)
    with pytest.raises(o.KernelError, match="float32 or bfloat16"):
        o.fp4_quantise(torch.zeros(4, 64, device="cuda", dtype=torch.float16), x)
    with pytest.raises(o.KernelError, match="contiguous values"):
        o.fp4_quantise(torch.zeros(64, 4, device="cuda").t(), x)
    with pytest.raises(o.KernelError, match="values"):
        o.fp4_quantise(torch.zeros(4, 64, device="cuda"), x, values=torch.zeros(4, 63, device="cuda"))
    with pytest.raises(o.KernelError, match="gate"):
        o.fp4_gated_product(x, w, o.fp4_rows(4, 16, "cuda"), st, activation="limited")
    with pytest.raises(o.KernelSizeError):
        o.fp4_gated_product(x, o.fp4_rows(36, 64, "cuda"), o.fp4_rows(4, 18, "cuda"), st)
    with pytest.raises(o.KernelSizeError):
        o.fp4_add_rmsnorm(torch.zeros(1, 32776, device="cuda"), None, torch.ones(32776, device="cuda"),
                          o.fp4_rows(1, 32776, "cuda"), 1e-6)
    with pytest.raises(o.KernelError, match="delta"):
        o.fp4_add_rmsnorm(torch.zeros(4, 64, device="cuda"), torch.zeros(3, 64, device="cuda"), torch.ones(64, device="cuda"), x, 1e-6)
    with pytest.raises(o.KernelSizeError):
        o.fp4_product(x, w, y, st, form="pair384")
    with pytest.raises(o.KernelSizeError):
        o.fp4_rows(2, 0, "cuda")
    assert int(st.item()) == 0


def test_a_refused_feed_forward_leaves_the_stream_alone():
    o, rows, width, inner = ops(), 3, 64, 40
    stream, delta, st = normal(rows, width, 1).cuda(), normal(rows, width, 2).cuda(), status()
    before, norm, y = stream.clone(), torch.ones(width, device="cuda"), torch.full((rows, width), 7.0, device="cuda")

    def off_by_eight(r):
        room = torch.zeros(r.codes.numel() + 16, dtype=torch.uint8, device="cuda")
        return o.Fp4Rows(room[8:8 + r.codes.numel()].view(r.codes.shape), r.scales, r.width)

    def scales_off_by_eight(r):
        room = torch.zeros(r.scales.numel() + 16, dtype=torch.uint8, device="cuda")
        return o.Fp4Rows(r.codes, room[8:8 + r.scales.numel()].view(r.scales.shape), r.width)

    def call(i=inner, change=None, which=None, **more):
        rows4 = [o.fp4_rows(2 * i, width, "cuda"), o.fp4_rows(width, i, "cuda"), o.fp4_rows(rows, width, "cuda"), o.fp4_rows(rows, i, "cuda")]
        if which is not None:
            rows4[which] = change(rows4[which])
        o.fp4_feed_forward(stream, delta, norm, 1e-6, *rows4, y, st, **more)

    with pytest.raises(o.KernelSizeError):
        call(12)
    for which in range(4):
        for change in (off_by_eight, scales_off_by_eight):
            with pytest.raises(o.KernelError, match="misaligned"):
                call(change=change, which=which)
    with pytest.raises(o.KernelError, match="gate"):
        call(activation="limited")
    with pytest.raises(o.KernelError, match="expected"):
        call(change=lambda r: o.fp4_rows(width, inner + 8, "cuda"), which=1)
    torch.cuda.synchronize()
    assert torch.equal(stream, before) and bool((y == 7).all()) and int(st.item()) == 0
    call()
    assert torch.equal(stream, before + delta)


@pytest.mark.parametrize("form", ["few", "pair192", "pair256", "pair384"])
@pytest.mark.parametrize("rows,features,width", [(3, 200, 3000), (600, 800, 1024)])
def test_a_wait_that_runs_out_is_given_up_cleanly(rows, features, width, form):
    o = ops()
    x, xv = held(normal(rows, width, 1))
    w, wv = held(normal(features, width, 2, False))
    y, st = torch.empty(rows, features, device="cuda", dtype=torch.bfloat16), status()
    try:
        o.set_wait_test(limit=1 << 14, drop_copy=1)
        o.fp4_product(x, w, y, st, form=form)
        torch.cuda.synchronize()
        word = int(st.item())
    finally:
        o.set_wait_test()
    assert word & 16, f"status {word}: the time-out bit is not set"
    st.zero_()
    o.fp4_product(x, w, y, st, form=form)
    assert int(st.item()) == 0
    want = xv @ wv.t()
    assert bool(((y.cpu().double() - want).abs() <= product_tolerance(xv, wv) + want.abs() * 2.0 ** -8).all())


@pytest.mark.parametrize("drop", [0, 1])
@pytest.mark.parametrize("rows,features,width", [(100, 512, 12288), (128, 1000, 4352), (70, 300, 2304), (200, 130, 8448)])
def test_sums_by_copies_are_given_up_cleanly(rows, features, width, drop):
    """Tiles whose sums go from block to block as copies, where all blocks give up or all but those with a single stage."""
    o = ops()
    x, xv = held(normal(rows, width, 1))
    w, wv = held(normal(features, width, 2, False))
    y, st = torch.empty(rows, features, device="cuda", dtype=torch.bfloat16), status()
    try:
        o.set_wait_test(limit=1 << 14, drop_copy=drop)
        o.fp4_product(x, w, y, st, form="few")
        torch.cuda.synchronize()
        word = int(st.item())
    finally:
        o.set_wait_test()
    assert word & 16, f"status {word}: the time-out bit is not set"
    st.zero_()
    want = xv @ wv.t()
    for _ in range(3):
        o.fp4_product(x, w, y, st, form="few")
        assert int(st.item()) == 0
        assert bool(((y.cpu().double() - want).abs() <= product_tolerance(xv, wv) + want.abs() * 2.0 ** -8).all())


@pytest.mark.parametrize("drop", [0, 1])
@pytest.mark.parametrize("rows,features,width", [(1, 208, 2816), (3, 208, 2816), (20, 144, 2816), (30, 48, 4352)])
def test_sums_by_stores_are_given_up_cleanly(rows, features, width, drop):
    """Tiles whose sums go from block to block as stores, where all blocks give up or all but one of a single stage, which sends its
    sums to blocks that wait for more and waits itself for what never comes."""
    o = ops()
    x, xv = held(normal(rows, width, 1))
    w, wv = held(normal(features, width, 2, False))
    y, a, st = torch.empty(rows, features, device="cuda"), o.fp4_rows(rows, features // 2, "cuda"), status()
    for call in (lambda: o.fp4_product(x, w, y, st, form="few"), lambda: o.fp4_gated_product(x, w, a, st, form="few")):
        try:
            o.set_wait_test(limit=1 << 14, drop_copy=drop)
            call()
            torch.cuda.synchronize()
            word = int(st.item())
        finally:
            o.set_wait_test()
        assert word & 16, f"status {word}: the time-out bit is not set"
        st.zero_()
    want, first = xv @ wv.t(), None
    for _ in range(3):
        o.fp4_product(x, w, y, st, form="few")
        o.fp4_gated_product(x, w, a, st, form="few")
        assert int(st.item()) == 0
        assert bool(((y.cpu().double() - want).abs() <= product_tolerance(xv, wv)).all())
        first = a.codes.clone() if first is None else first
        assert torch.equal(a.codes, first)


# ---------------------------------------------------------------- a model whose feed-forwards are held so
def plain_mlp(x, w, prefix):
    """The feed-forward of the plain model with weights and activations rounded."""
    h = plain.rounded(x.double())
    gate = h @ plain.rounded(w[f"{prefix}.gate_proj.weight"].double()).t()
    up = h @ plain.rounded(w[f"{prefix}.up_proj.weight"].double()).t()
    a = plain.rounded(gate * torch.sigmoid(gate) * up)
    return (a @ plain.rounded(w[f"{prefix}.down_proj.weight"].double()).t()).to(x.dtype)


@pytest.mark.parametrize("key", ["a", "b", "d"])
def test_model_with_fp4_feed_forwards(tiny_folders, monkeypatch, key):
    """In float32, prompts whole and token by token.  The engine's float32 sums differ from the plain model's by about 1e-6, which
    moves a value across a boundary between two codes once in some 10^5 of them (a test has 10^4) and nothing else by more than the
    1e-5 of the float32 replays; a moved code would show as 1e-3 and more of the logits, so a tenth of that is the bound."""
    import plain_qwen3
    from conftest import TINY, random_tokens
    from qwen3_from_scratch_b200.engine.batch import Entry
    from qwen3_from_scratch_b200.engine.session import Session
    folder = tiny_folders[key]
    cfg, w = plain_qwen3.read_model_folder(folder)
    ids = random_tokens(TINY[key][0]["vocab_size"], 20, 3)
    without = plain_qwen3.forward_logits(cfg, w, ids)
    monkeypatch.setattr(plain_qwen3, "swiglu_mlp", plain_mlp)
    want = plain_qwen3.forward_logits(cfg, w, ids).double()
    session = Session(folder, dtype="float32", page_size=8, num_pages=16, max_seqs=2, max_step_tokens=64, feed_forward_weights="fp4")
    whole = session.step([Entry("r", ids, list(range(20)))]).cpu().double()
    session.end("r")
    rows = [session.step([Entry("s", [t], [0])]).cpu().double() for t in ids]
    session.check_status()
    scale = float(want.abs().max())
    for got in (whole, torch.cat(rows)):
        assert float((got - want).abs().max()) <= 1e-4 * scale
    assert float((without.double() - want).abs().max()) > 1e-3 * scale  # the rounding is seen at all


def test_engine_generates_with_fp4_feed_forwards(tiny_folders):
    from qwen3_from_scratch_b200.engine.engine import SyncEngine
    engine = SyncEngine(tiny_folders["d"], max_num_seqs=4, max_num_tokens=256, num_pages=64, max_new_tokens=12,
                        feed_forward_weights="fp4")
    first = [r.token_ids for r in engine.batch_generate([[1, 2, 3], list(range(5, 150))], ignore_eos=True)[0]]
    again = [r.token_ids for r in engine.batch_generate([[1, 2, 3], list(range(5, 150))], ignore_eos=True)[0]]
    assert first == again and [len(t) for t in first] == [12, 12]
    with pytest.raises(ValueError, match="fp4"):
        SyncEngine(tiny_folders["d"], num_pages=64, feed_forward_weights="int3")


# ---------------------------------------------------------------- codes and scales as arithmetic on bytes leaves them
@pytest.mark.parametrize("wide", [torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("rows,inner,width", [(3, 40, 264), (300, 72, 128)])
def test_products_of_bytes_in_a_wider_integer_type(rows, inner, width, wide):
    o = ops()
    x, gu = held(normal(rows, width, 1))[0], held(interleaved(normal(inner, width, 2, False), normal(inner, width, 3, False)))[0]
    down = held(normal(width, inner, 4, False))[0]
    as_wide = [o.Fp4Rows(r.codes.to(wide), r.scales.to(wide), r.width) for r in (x, gu, down)]
    st, y, y2 = status(), torch.empty(rows, 2 * inner, device="cuda"), torch.empty(rows, 2 * inner, device="cuda")
    o.fp4_product(x, gu, y, st)
    o.fp4_product(as_wide[0], as_wide[1], y2, st)
    assert torch.equal(y, y2)
    a, a2 = o.fp4_rows(rows, inner, "cuda"), o.fp4_rows(rows, inner, "cuda")
    o.fp4_gated_product(x, gu, a, st)
    o.fp4_gated_product(as_wide[0], as_wide[1], a2, st)
    assert torch.equal(a.codes, a2.codes)
    stream, norm, h = normal(rows, width, 5).cuda(), torch.ones(width, device="cuda"), o.fp4_rows(rows, width, "cuda")
    z, z2 = torch.empty(rows, width, device="cuda"), torch.empty(rows, width, device="cuda")
    o.fp4_feed_forward(stream, None, norm, 1e-6, gu, down, h, a, z, st)
    o.fp4_feed_forward(stream, None, norm, 1e-6, as_wide[1], as_wide[2], h, a2, z2, st)
    assert torch.equal(z, z2) and int(st.item()) == 0
    # what a call writes has to be bytes, and what it reads has to be whole numbers
    with pytest.raises(o.KernelError, match="uint8"):
        o.fp4_quantise(stream, o.Fp4Rows(h.codes.to(wide), h.scales, width))
    with pytest.raises(o.KernelError, match="uint8"):
        o.fp4_gated_product(x, gu, o.Fp4Rows(a.codes.to(wide), a.scales, inner), st)
    with pytest.raises(o.KernelError, match="uint8"):
        o.fp4_product(o.Fp4Rows(x.codes.float(), x.scales, width), gu, y, st)


def test_feed_forward_of_a_prompt_is_its_parts():
    """Where the rule takes pairs of CTAs for both products, several tiles each."""
    for dtype in DT:
        test_feed_forward_is_its_parts(dtype, 2100, 1024, 4104)


# ---------------------------------------------------------------- models in bfloat16 and behind other norms
def rms(t):
    return float(t.double().square().mean().sqrt())


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("key", ["a", "b", "d"])
def test_model_with_fp4_feed_forwards_in_bfloat16(tiny_folders, monkeypatch, key, graphs):
    """The logits of a prompt and of single tokens, whole against whole.  Rounding to bfloat16 moves values across boundaries between
    codes, so single logits may be off by a code's step; what is held is the root mean square over 60 positions, to 1.5 times what such
    rounding does in the plain model (operands and results of the attention's projections, rotated heads, the feed-forward's result and
    the head's operand).  A model without the rounding to four bits is further off than that."""
    import plain_qwen3
    from conftest import TINY, random_tokens
    from qwen3_from_scratch_b200.engine.batch import Entry
    from qwen3_from_scratch_b200.engine.session import Session
    folder = tiny_folders[key]
    cfg, w = plain_qwen3.read_model_folder(folder)
    ids = random_tokens(TINY[key][0]["vocab_size"], 60, 3)
    without = plain_qwen3.forward_logits(cfg, w, ids)
    monkeypatch.setattr(plain_qwen3, "swiglu_mlp", plain_mlp)
    want = plain_qwen3.forward_logits(cfg, w, ids)

    def cut(t):
        return t.to(torch.bfloat16).to(t.dtype)

    rope, attend, mixer, head = (getattr(plain_qwen3, n) for n in ("apply_rope", "causal_attention", "self_attention", "lm_head"))
    with monkeypatch.context() as m:
        m.setattr(plain_qwen3, "apply_rope", lambda x, c, s: cut(rope(cut(x), c, s)))
        m.setattr(plain_qwen3, "causal_attention", lambda q, k, v, window=None: cut(attend(q, k, cut(v), window)))
        m.setattr(plain_qwen3, "self_attention", lambda x, *rest: cut(mixer(cut(x), *rest)))
        m.setattr(plain_qwen3, "swiglu_mlp", lambda *rest: cut(plain_mlp(*rest)))
        m.setattr(plain_qwen3, "lm_head", lambda h, *rest: head(cut(h), *rest))
        noisy = plain_qwen3.forward_logits(cfg, w, ids)
    bound = 1.5 * rms(noisy - want)
    assert bound < 0.85 * rms(without - want)
    session = Session(folder, dtype="bfloat16", page_size=16, num_pages=24, max_seqs=2, max_step_tokens=64, cuda_graphs=graphs,
                      feed_forward_weights="fp4")
    whole = session.step([Entry("r", ids, list(range(60)))]).float().cpu()
    session.end("r")
    rows = [session.step([Entry("s", [t], [0])]).float().cpu().clone() for t in ids]
    session.check_status()
    assert rms(whole - want) <= bound and rms(torch.cat(rows) - want) <= bound


@pytest.mark.parametrize("key", ["a", "d"])
def test_model_whose_feed_forwards_read_a_normed_sum(tiny_folders, monkeypatch, key):
    """A block whose mixer leaves several terms norms them before the feed-forward, which then rounds the normed rows: in float32 the
    logits of the same bound as above."""
    import plain_qwen3
    from conftest import TINY, random_tokens
    from qwen3_from_scratch_b200.engine.batch import Entry
    from qwen3_from_scratch_b200.engine.session import Session
    from qwen3_from_scratch_b200.parts.base import PendingSum
    from qwen3_from_scratch_b200.parts.mlp import GatedMLP
    folder = tiny_folders[key]
    cfg, w = plain_qwen3.read_model_folder(folder)
    ids = random_tokens(TINY[key][0]["vocab_size"], 20, 3)
    monkeypatch.setattr(plain_qwen3, "swiglu_mlp", plain_mlp)
    want = plain_qwen3.forward_logits(cfg, w, ids).double()
    session = Session(folder, dtype="float32", page_size=8, num_pages=16, max_seqs=2, max_step_tokens=64, feed_forward_weights="fp4",
                      cuda_graphs=False)
    for block in session.model.layers:
        def two_terms(*args, forward=block.mixer.forward, **more):
            a = forward(*args, **more)
            return PendingSum.of(a, torch.zeros_like(a))
        monkeypatch.setattr(block.mixer, "forward", two_terms)
    calls = []
    inner = GatedMLP._forward_fp4
    monkeypatch.setattr(GatedMLP, "_forward_fp4", lambda self, x: calls.append(0) or inner(self, x))
    whole = session.step([Entry("r", ids, list(range(20)))]).cpu().double()
    session.end("r")
    rows = [session.step([Entry("s", [t], [0])]).cpu().double() for t in ids]
    session.check_status()
    assert len(calls) == len(session.model.layers) * 21
    for got in (whole, torch.cat(rows)):
        assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max())


def plain_relu_glu(x, w, p):
    """The feed-forward of the plain Binupel with weights and activations rounded."""
    h = plain.rounded(x)
    a = plain.rounded(torch.relu(h @ plain.rounded(w[p + "gate"]).t()) * (h @ plain.rounded(w[p + "up"]).t()))
    return a @ plain.rounded(w[p + "down"]).t()


@pytest.mark.parametrize("key", ["p", "q", "r"])
def test_post_norm_model_with_fp4_feed_forwards(tmp_path, monkeypatch, key):
    """Binupel, whose norms stand behind the sums and whose gates are ReLU: float32, a prompt whole and token by token.  In the plain
    model a disturbance of 2e-6 of the embeddings moves no code at these tokens (six drawn), so the bound is that of the model above."""
    import plain_binupel
    from binupel_models import CONFIGS, make_folder
    from qwen3_from_scratch_b200.engine.batch import Entry
    from qwen3_from_scratch_b200.engine.session import Session
    folder = make_folder(str(tmp_path), *CONFIGS[key])
    cfg, w = plain_binupel.read_model_folder(folder)
    ids = torch.randint(0, cfg["vocab"], (20,), generator=torch.Generator().manual_seed(3)).tolist()
    without = plain_binupel.forward_logits(cfg, w, ids)
    monkeypatch.setattr(plain_binupel, "relu_glu", plain_relu_glu)
    want = plain_binupel.forward_logits(cfg, w, ids)
    session = Session(folder, dtype="float32", page_size=8, num_pages=16, max_seqs=2, max_step_tokens=64, feed_forward_weights="fp4")
    whole = session.step([Entry("r", ids, list(range(20)))]).cpu().double()
    session.end("r")
    rows = [session.step([Entry("s", [t], [0])]).cpu().double() for t in ids]
    session.check_status()
    scale = float(want.abs().max())
    for got in (whole, torch.cat(rows)):
        assert float((got - want).abs().max()) <= 1e-4 * scale
    assert float((without - want).abs().max()) > 1e-3 * scale


@pytest.mark.parametrize("act", ["silu", "relu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_gated_feed_forward_of_normed_rows(rows, dtype, act):
    """The part by itself, given rows that are normed already: every result is a sum of what the gate may have left (both ends of each
    value's range) times the weight, rounded once."""
    from qwen3_from_scratch_b200.parts.base import PartSpec, Runtime
    from qwen3_from_scratch_b200.registry import create_part
    width, inner = 136, 264
    part = create_part("feed_forward", PartSpec("gated_mlp", {"hidden_size": width, "intermediate_size": inner, "activation": act}), name="f")
    g = torch.Generator().manual_seed(4)
    stored = {n: (torch.randn(s, generator=g) * s[1] ** -0.5).to(torch.bfloat16)
              for n, s in (("gate", (inner, width)), ("up", (inner, width)), ("down", (width, inner)))}
    x = normal(rows, width, rows).to(DT[dtype])
    rt = Runtime(torch.device("cuda:0"), DT[dtype], 320, 2, feed_forward_weights="fp4")
    part.setup(rt, {f"f.{n}_proj.weight": t.to(DT[dtype]).cuda() for n, t in stored.items()})
    got = part.forward(x.cuda()).cpu()
    assert got.dtype == DT[dtype] and got.shape == x.shape and int(rt.status.item()) == 0
    gate, up, down = (plain.rounded(stored[n].double()) for n in ("gate", "up", "down"))
    a, slack = gated_bounds(plain.rounded(x.double()), interleaved(gate, up), act)
    low, high = plain.between(a, slack)
    middle, reach = (low + high) / 2, (high - low) / 2
    want, tol = middle @ down.t(), reach @ down.abs().t() + product_tolerance(middle.abs() + reach, down)
    if dtype == "bfloat16":
        tol = tol + (want.abs() + tol) * 2.0 ** -8
    assert bool(((got.double() - want).abs() <= tol).all())
    assert float((reach > 0).double().mean()) < 0.01  # the ranges hardly ever hold two values


# ---------------------------------------------------------------- the stream that every operator asks for
def test_the_stream_handle_is_torchs_current_one():
    import threading
    o, side = ops(), torch.cuda.Stream()
    torch.zeros(1, device="cuda")
    assert o._stream() == torch.cuda.current_stream().cuda_stream
    with torch.cuda.stream(side):
        assert o._stream() == side.cuda_stream == torch.cuda.current_stream().cuda_stream
        seen = []
        thread = threading.Thread(target=lambda: seen.append((o._stream(), torch.cuda.current_stream().cuda_stream)))
        thread.start()
        thread.join()
        assert len(seen) == 1 and seen[0][0] == seen[0][1]
    assert o._stream() == torch.cuda.current_stream().cuda_stream != side.cuda_stream
