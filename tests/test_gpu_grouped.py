"""Row groups and grouped linear maps on the GPU against their definition in 64 bits on the CPU."""
import gc

import numpy as np
import pytest
import torch

import openequivariance_b200 as oeq
from openequivariance_b200 import Irreps
import grouped_reference as ref
from conftest import ROOT

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def no_wait_was_abandoned():
    yield
    oeq.GroupedLinear.check_device_status()


def host(t):
    return t.detach().cpu().numpy()


# ------------------------------------------------------------------------------------------ row groups

def check_groups(index, groups):
    got = oeq.RowGroups(torch.from_numpy(index).cuda(), groups)
    for name, want in zip(("order", "slots", "offsets", "blocks"), ref.row_groups(index, groups)):
        np.testing.assert_array_equal(host(getattr(got, name)), want, err_msg=name)
    assert got.rows == len(index) and got.num_groups == groups


@pytest.mark.parametrize("groups", [1, 2, 10, 89, 1500, 8191])
@pytest.mark.parametrize("rows", [0, 1, 27, 31, 32, 33, 1000, 8192, 8193, 40961])
def test_row_groups(rows, groups):
    rng = np.random.default_rng(rows + groups)
    check_groups(rng.integers(-1, groups, rows), groups)


@pytest.mark.parametrize("rows", [500, 20011])
@pytest.mark.parametrize("kind", ["one", "none", "sorted", "reversed", "outside", "last"])
def test_row_groups_of_one_shape(kind, rows):
    rng, groups = np.random.default_rng(3), 37
    index = rng.integers(0, groups, rows)
    if kind == "one":
        index[:] = 17
    elif kind == "none":
        index[:] = -1
    elif kind == "sorted":
        index.sort()
    elif kind == "reversed":
        index = np.sort(index)[::-1].copy()
    elif kind == "outside":                 # every value that is no group: they keep their order at the end
        index = rng.choice(np.array([-2 ** 62, -1, 37, 38, 2 ** 31, 2 ** 32 + 5, 2 ** 62, 3, 36]), rows)
    else:
        index[:] = groups - 1
    check_groups(index, groups)


def test_row_groups_many():
    check_groups(np.random.default_rng(5).zipf(1.3, 1_000_003) - 1, 1999)


def test_row_groups_of_a_strided_index():
    wide = torch.randint(0, 9, (700, 3), device="cuda")
    got, want = oeq.RowGroups(wide[:, 1], 9), oeq.RowGroups(wide[:, 1].contiguous(), 9)
    assert torch.equal(got.order, want.order) and torch.equal(got.blocks, want.blocks)


@pytest.mark.parametrize("rows,counts", [
    (0, [0]), (0, [3]), (5, [5]), (5, [2]), (5, [0, 0, 5, 0]), (5, [9, 1]), (64, [64]), (65, [1, 64]), (10, [-4, 3, -1, 4]),
    (1000, [2 ** 62, 2 ** 62]), (1000, [500, 2 ** 40, 7])])
def test_row_groups_from_counts(rows, counts):
    check_counts(rows, np.array(counts, dtype=np.int64))


@pytest.mark.parametrize("groups,mean", [(1, 100), (512, 3), (513, 40), (1000, 50), (8191, 1), (8191, 30)])
def test_row_groups_from_many_counts(groups, mean):
    rng = np.random.default_rng(groups)
    counts = rng.integers(0, 2 * mean + 1, groups)
    for rows in {int(counts.sum()), int(counts.sum()) + 77, int(counts.sum()) * 2 // 3}:
        check_counts(rows, counts)


def check_counts(rows, counts):
    got = oeq.RowGroups.from_counts(torch.from_numpy(counts).cuda(), rows)
    for name, want in zip(("index", "offsets", "blocks"), ref.from_counts(counts.tolist(), rows)):
        np.testing.assert_array_equal(host(getattr(got, name)), want, err_msg=name)
    assert got.order is None and got.slots is None


# ------------------------------------------------------------------------------------------ linear maps

def inputs(irreps_in, irreps_out, dtype, rows, groups, seed, by="index", without=0.1):
    """x, w, dz, index on the CPU in float64, with the values that the type has."""
    gen = torch.Generator().manual_seed(seed)
    numel = oeq.GroupedLinear(irreps_in, irreps_out).weight_numel
    draw = lambda *shape: torch.randn(*shape, generator=gen, dtype=torch.float64).to(dtype).double()
    index = torch.randint(0, groups, (rows,), generator=gen)
    index[torch.rand(rows, generator=gen) < without] = -1
    if by == "counts":
        index = torch.cat([index[index >= 0].sort().values, index[index < 0]])
    return draw(rows, Irreps(irreps_in).dim), draw(groups, numel), draw(rows, Irreps(irreps_out).dim), index


def groups_of(index, groups, by="index"):
    if by == "counts":
        return oeq.RowGroups.from_counts(torch.bincount(index[index >= 0], minlength=groups).cuda(), len(index))
    return oeq.RowGroups(index.cuda(), groups)


def check_linear(irreps_in, irreps_out, dtype, rows, groups, seed=0, by="index", without=0.1, change=lambda t: t):
    x, w, dz, index = inputs(irreps_in, irreps_out, dtype, rows, groups, seed, by, without)
    lin = oeq.GroupedLinear(irreps_in, irreps_out)
    plan = groups_of(index, groups, by)
    xg, wg, dzg = (change(t.to(dtype).cuda()).requires_grad_(True) for t in (x, w, dz))
    z = lin(xg, wg, plan)
    dx, dw = torch.autograd.grad(z, (xg, wg), dzg)
    compare(irreps_in, irreps_out, dtype, x, w, dz, index, z, dx, dw)


def compare(irreps_in, irreps_out, dtype, x, w, dz, index, z, dx, dw):
    want = ref.linear(irreps_in, irreps_out, x, w, index, dz)
    size = ref.linear(irreps_in, irreps_out, x.abs(), w.abs(), index, dz.abs())
    a, b = Irreps(irreps_in), Irreps(irreps_out)
    most = max([ir.dim for _, ir in a] + [1]) * int(torch.bincount(index[index >= 0], minlength=1).max() if len(index) else 0)
    terms = (sum(m for m, _ in a), sum(m for m, _ in b), most)
    for name, got, t, s, n in zip(("z", "dx", "dw"), (z, dx, dw), want, size, terms):
        assert got.dtype == dtype and got.shape == t.shape
        got = got.detach().cpu().double()
        over = (got - t).abs() - ref.allowed(dtype, t, s, n)
        assert bool((over <= 0).all()), f"{name}: {float(over.max())} over, at {int(over.argmax())}"
        if dtype in (F32, F64) and t.numel() and float(t.abs().max()) > 0:          # and the parity bound of this repository's kernels
            assert float((got - t).abs().max() / t.abs().max()) < (1e-5 if dtype == F32 else 1e-12), name


TYPES = [F32, F64, BF16, F16]
TYPE_IDS = ["f32", "f64", "bf16", "f16"]


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("irreps_in,irreps_out", [
    ("16x0e", "16x0e"),
    ("128x0e+128x1o+128x2e", "128x0e+128x1o+128x2e"),
    ("33x0e+17x1o+5x2e+3x2o", "19x0e+40x0e+21x1o+6x2e"),
    ("32x0e+32x0e+7x1o", "1x0e+130x0e+65x1o+4x3o"),
    ("3x3o+2x4e+1x5o", "5x3o+9x4e+2x5o"),
    ("1x0e", "1x0e"),
    ("200x0e", "264x0e"),
    ("8x1o", "8x1e")], ids=["scalars", "wide", "odd", "joined", "high", "one", "long", "nothing"])
def test_linear(irreps_in, irreps_out, dtype):
    check_linear(irreps_in, irreps_out, dtype, 211, 7, seed=1)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("irreps_in,irreps_out", [("1100x0e", "300x0e"), ("300x0e", "1100x0e"), ("520x0e+8x1o", "136x0e+272x1o"), ("600x1o", "40x1o")])
def test_linear_of_many_channels(irreps_in, irreps_out, dtype):
    """Weights of a group that do not fit shared memory, several tiles of channels."""
    check_linear(irreps_in, irreps_out, dtype, 300, 3, seed=3)


CHAIN = 32          # additions to an accumulator: 256 channels, eight an addition


@pytest.mark.parametrize("irreps,other", [("256x0e", "80x0e"), ("264x0e", "16x0e"), ("2048x0e", "48x0e"), ("4096x0e", "80x0e"), ("4096x0e", "33x0e"), ("2047x0e", "160x0e"),
                                          ("1024x0e+512x0e+2048x0e+7x0e", "40x0e"), ("1500x1o", "24x1o"), ("1100x2e+1024x3o", "72x2e+8x3o")])
def test_float32_sums_over_many_channels(irreps, other):
    """The error of a sum does not grow with the number of its terms, in the product (many channels in) and in dX (many channels out)."""
    rows, groups = 150, 2
    for names in ((irreps, other), (other, irreps)):
        x, w, dz, index = inputs(*names, F32, rows, groups, 21)
        lin = oeq.GroupedLinear(*names)
        xg, wg, dzg = (t.float().cuda().requires_grad_(True) for t in (x, w, dz))
        z = lin(xg, wg, groups_of(index, groups))
        dx, = torch.autograd.grad(z, xg, dzg)
        want_z, want_dx, _ = ref.linear(*names, x, w, index, dz)
        got, want, a = (z, want_z, names[0]) if names[0] == irreps else (dx, want_dx, names[1])
        for (_, ir), block in zip(Irreps(other), Irreps(other).slices()):           # (they have different numbers of terms)
            terms = sum(m for m, of in Irreps(a) if of == ir)
            e = got.detach().cpu().double()[:, block] - want[:, block]
            short = float(e.norm() / want[:, block].norm())
            assert short <= ref.allowed_norm(CHAIN, -(-terms // (8 * CHAIN))), (names, short)
            assert float(e.abs().max() / want[:, block].abs().max()) < 1e-5


def test_float32_sums_over_many_channels_of_many_rows():
    """Several tiles of rows in each range, an odd number of chunks of results; every run the same."""
    names, rows, groups = ("700x0e+300x1o", "136x0e+40x1o"), 20_000, 3
    x, w, dz, index = inputs(*names, F32, rows, groups, 22)
    lin, plan = oeq.GroupedLinear(*names), groups_of(index, groups)
    xg, wg, dzg = (t.float().cuda().requires_grad_(True) for t in (x, w, dz))
    z = lin(xg, wg, plan)
    dx, dw = torch.autograd.grad(z, (xg, wg), dzg)
    compare(*names, F32, x, w, dz, index, z, dx, dw)
    for _ in range(2):
        assert torch.equal(lin(xg, wg, plan), z)


@pytest.mark.parametrize("irreps,rows", [("64x0e", 400_000), ("32x3o", 60_000), ("1400x0e", 30_000)])
def test_float32_weight_gradients_of_many_rows(irreps, rows):
    """A sum over all rows, in many ranges and in one (a tile for each CTA)."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    lin, (mul, ir) = oeq.GroupedLinear(irreps, irreps), Irreps(irreps)[0]
    x, dz = (torch.randn(rows, mul * ir.dim, device="cuda", generator=gen) for _ in range(2))
    w = torch.zeros(1, mul * mul, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(lin(x, w, oeq.RowGroups(torch.zeros(rows, dtype=torch.int64, device="cuda"), 1)), w, dz)
    left, right = (t.view(rows, mul, ir.dim).transpose(1, 2).reshape(rows * ir.dim, mul).double() for t in (x, dz))
    want = left.T @ right / mul ** 0.5
    # (a chain ends with a unit of rows of all components: 35 additions of eight rows at most)
    assert float((dw.double().view(mul, mul) - want).norm() / want.norm()) <= ref.allowed_norm(35, -(-rows * ir.dim // 256))


@pytest.mark.parametrize("irreps_in,irreps_out,rows", [("1600x4e", "1600x4e", 4000), ("64x4e", "48x4e", 50_000), ("9000x4e", "40x4e", 64)])
def test_float32_sums_of_high_degrees(irreps_in, irreps_out, rows):
    """The FMA kernels: long sums of a weight gradient in one range of rows and in many, and of a product."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    lin, a, b = oeq.GroupedLinear(irreps_in, irreps_out), Irreps(irreps_in)[0].mul, Irreps(irreps_out)[0].mul
    x, dz = (torch.randn(rows, m * 9, device="cuda", generator=gen) for m in (a, b))
    w = torch.randn(1, a * b, device="cuda", generator=gen).requires_grad_(True)
    z = lin(x, w, oeq.RowGroups(torch.zeros(rows, dtype=torch.int64, device="cuda"), 1))
    dw, = torch.autograd.grad(z, w, dz)
    left, right = (t.double().view(rows, -1, 9).transpose(1, 2).reshape(rows * 9, -1) for t in (x, dz))
    for got, want, terms in ((z.detach().double().view(rows, b, 9).transpose(1, 2).reshape(rows * 9, b), left @ w.detach().double().view(a, b) / a ** 0.5, a),
                             (dw.double().view(a, b), left.T @ right / a ** 0.5, rows * 9)):
        assert float((got - want).norm() / want.norm()) <= ref.allowed_norm_rounded(min(terms, 512), -(-terms // 512))


@pytest.mark.parametrize("irreps,dtype", [("4200000x0e", F64), ("40000x64e", F32)])
def test_more_columns_of_results_than_a_grid_has(irreps, dtype):
    """Over 65 535 pieces of 64 channels and one component, with rows that have no group."""
    one = "1x" + irreps.split("x")[1]
    check_linear(one, irreps, dtype, 5, 2, seed=5, without=0.4)


def test_blocks_without_a_path():
    """Irreps that one side alone has, of any degree, and blocks of no channels: zeros, with and without gradients."""
    for names in (("4x0e+2x6e", "3x9o+4x0e"), ("0x1o+4x0e+0x0e", "0x0e+8x0e+0x2e"), ("2x5e", "2x5o")):
        for dtype in (F32, F64, BF16):
            check_linear(*names, dtype, 70, 3, seed=1)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_expanded_gradients(dtype):
    """The gradient that a sum sends back has one value for all."""
    x, w, _, index = inputs("16x0e+8x1o", "8x0e+8x1o", dtype, 120, 4, 2)
    lin, plan = oeq.GroupedLinear("16x0e+8x1o", "8x0e+8x1o"), groups_of(index, 4)
    xg, wg = (t.to(dtype).cuda().requires_grad_(True) for t in (x, w))
    z = lin(xg, wg, plan)
    z.sum().backward()
    compare("16x0e+8x1o", "8x0e+8x1o", dtype, x, w, torch.ones(z.shape, dtype=F64), index, z, xg.grad, wg.grad)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 127, 128, 129, 700])
def test_linear_rows(rows, dtype):
    check_linear("32x0e+20x1o", "24x0e+32x1o", dtype, rows, 3, seed=rows)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("groups", [1, 2, 300, 8191])
def test_linear_groups(groups, dtype):
    check_linear("8x0e+4x1o", "12x0e+4x1o", dtype, 1500, groups, seed=groups)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("without", [0.0, 0.5, 1.0])
def test_linear_of_counts(without, dtype):
    check_linear("40x0e+16x1o+8x2e", "24x0e+24x1o+8x2e", dtype, 901, 11, seed=4, by="counts", without=without)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_linear_of_few_long_groups(dtype):
    """Sums over many rows, parts of a group from many ranges of rows."""
    check_linear("64x0e+16x1o", "48x0e+16x1o", dtype, 9001, 2, seed=8, without=0.0)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_no_rows(dtype):
    lin = oeq.GroupedLinear("4x0e", "5x0e")
    x, w = torch.zeros(0, 4, device="cuda", dtype=dtype, requires_grad=True), torch.ones(3, 20, device="cuda", dtype=dtype, requires_grad=True)
    for plan in (oeq.RowGroups(torch.zeros(0, dtype=torch.int64, device="cuda"), 3),
                 oeq.RowGroups.from_counts(torch.zeros(3, dtype=torch.int64, device="cuda"), 0)):
        z = lin(x, w, plan)
        dx, dw = torch.autograd.grad(z, (x, w), torch.zeros_like(z))
        assert z.shape == (0, 5) and dx.shape == x.shape and not dw.any()


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_strided_and_unaligned_tensors(dtype):
    def wider(t):
        out = torch.full((t.shape[0], t.shape[1] + 3), 7.0, dtype=t.dtype, device=t.device)
        out[:, 1:-2] = t
        return out[:, 1:-2].detach()

    def shifted(t):
        out = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view_as(t)
        return out.copy_(t).detach()

    for change in (wider, shifted, lambda t: t.t().contiguous().t().detach()):
        check_linear("16x0e+8x1o", "32x0e+8x1o", dtype, 150, 4, seed=2, change=change)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_every_row_of_the_results_is_written(dtype):
    """Memory that held NaN: rows without a group, groups without rows, output blocks without a path."""
    x, w, dz, index = inputs("8x0e+3x1o", "8x0e+3x1e", dtype, 300, 5, 6, without=0.4)
    index[index == 2] = 3
    plan = groups_of(index, 5)
    lin = oeq.GroupedLinear("8x0e+3x1o", "8x0e+3x1e")
    for _ in range(3):
        junk = [torch.full((300, 17), float("nan"), dtype=dtype, device="cuda") for _ in range(4)] + \
               [torch.full((5, 64), float("nan"), dtype=dtype, device="cuda") for _ in range(4)]
        del junk
        xg, wg = (t.to(dtype).cuda().requires_grad_(True) for t in (x, w))
        z = lin(xg, wg, plan)
        dx, dw = torch.autograd.grad(z, (xg, wg), dz.to(dtype).cuda())
        compare("8x0e+3x1o", "8x0e+3x1e", dtype, x, w, dz, index, z, dx, dw)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_values_that_are_not_numbers_stay_in_their_rows(dtype):
    x, w, dz, index = inputs("64x0e+8x1o", "48x0e+8x1o", dtype, 400, 6, 9, without=0.2)
    bad = torch.zeros(400, dtype=torch.bool)
    bad[[0, 17, 18, 200, 399]] = True
    index[17] = -1                                                  # in a row without a group: nowhere
    xb, wb = x.clone(), w.clone()
    xb[bad] = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=torch.float64)[torch.arange(int(bad.sum())) % 3][:, None]
    wb[4] = float("nan")
    lin, plan = oeq.GroupedLinear("64x0e+8x1o", "48x0e+8x1o"), groups_of(index, 6)
    clean = lin(x.to(dtype).cuda(), w.to(dtype).cuda(), plan).cpu()
    z = lin(xb.to(dtype).cuda(), wb.to(dtype).cuda(), plan).cpu()
    touched = (bad & (index >= 0)) | (index == 4)
    assert torch.equal(z[~touched], clean[~touched])
    assert not torch.isfinite(z[touched]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("names", [("64x0e+8x1o+6x2e", "48x0e+8x1o+6x2e"), ("64x0e+16x1o+8x3o", "32x0e+64x1o+8x3o"), ("5x0e+2x4e", "7x0e+2x4e")], ids=["odd", "aligned", "high"])
def test_gradients_of_values_that_are_not_numbers_stay_in_their_rows_and_groups(names, dtype):
    """Rows of a product and of dX have their own; a row's numbers reach the weight gradient of its group alone, and a row without a
    group reaches none."""
    x, w, dz, index = inputs(*names, dtype, 400, 6, 19, without=0.2)
    index[index == 4] = 1                                           # a group without rows
    bad = torch.zeros(400, dtype=torch.bool)
    bad[[0, 17, 18, 399]] = True
    index[bad] = torch.tensor([2, -1, 5, 2])
    value = torch.tensor([float("nan"), float("inf"), -float("inf"), float("nan")], dtype=F64)[:, None]
    xb, dzb = x.clone(), dz.clone()
    xb[bad], dzb[bad] = value, value
    lin, plan = oeq.GroupedLinear(*names), groups_of(index, 6)

    def gradients(x, dz):
        a, b = (t.to(dtype).cuda().requires_grad_(True) for t in (x, w))
        return [t.cpu() for t in torch.autograd.grad(lin(a, b, plan), (a, b), dz.to(dtype).cuda())]

    clean_dx, clean_dw = gradients(x, dz)
    touched, kept = bad & (index >= 0), [0, 1, 3, 4]
    for dx, dw in (gradients(xb, dz), gradients(x, dzb)):
        assert torch.equal(dw[kept], clean_dw[kept]) and not dw[4].any()
        assert not torch.isfinite(dw[[2, 5]]).any()
    assert torch.equal(gradients(xb, dz)[0], clean_dx)
    dx = gradients(x, dzb)[0]
    assert torch.equal(dx[~touched], clean_dx[~touched]) and not torch.isfinite(dx[touched]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("names", [("128x0e+128x1o+64x2e+1x4e", "128x0e+64x1o+128x2e+1x4e"), ("64x0e+5x2e+64x1o", "64x0e+5x2e+64x1o")], ids=["high", "odd"])
def test_wide_blocks_beside_one_that_takes_another_way(names, dtype):
    check_linear(*names, dtype, 700, 5, seed=6)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_linear_of_many_channels_and_rows(dtype):
    """Weights that do not stay in shared memory, many tiles of rows in a CTA's range, many groups in it."""
    check_linear("520x0e+136x1o", "600x0e+136x1o", dtype, 6001, 40, seed=9)


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_the_same_result_in_every_run(dtype):
    x, w, dz, index = inputs("64x0e+32x1o", "64x0e+32x1o", dtype, 6001, 5, 3)
    plan, lin = groups_of(index, 5), oeq.GroupedLinear("64x0e+32x1o", "64x0e+32x1o")
    runs = []
    for _ in range(3):
        xg, wg = (t.to(dtype).cuda().requires_grad_(True) for t in (x, w))
        z = lin(xg, wg, plan)
        runs.append((z.detach(), *torch.autograd.grad(z, (xg, wg), dz.to(dtype).cuda())))
    for run in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(run, runs[0]))


def test_gradients_against_differences():
    x, w, dz, index = inputs("3x0e+2x1o", "2x0e+2x1o", F64, 9, 3, 5)
    plan, lin = groups_of(index, 3), oeq.GroupedLinear("3x0e+2x1o", "2x0e+2x1o")
    x, w = (t.cuda().requires_grad_(True) for t in (x, w))
    call = lambda p, q: lin(p, q, plan)
    assert torch.autograd.gradcheck(call, (x, w))
    assert torch.autograd.gradgradcheck(call, (x, w))


@pytest.mark.parametrize("dtype", [F32, F64], ids=["f32", "f64"])
def test_second_derivatives(dtype):
    """Derivatives of <ex, dX> + <ew, dW>, as a training step on forces takes them."""
    names = "24x0e+16x1o", "40x0e+8x1o"
    x, w, dz, index = inputs(*names, dtype, 333, 4, 12)
    ex, ew, _, _ = inputs(*names, dtype, 333, 4, 13)
    plan, lin = groups_of(index, 4), oeq.GroupedLinear(*names)
    xg, wg, dzg = (t.to(dtype).cuda().requires_grad_(True) for t in (x, w, dz))
    first = torch.autograd.grad(lin(xg, wg, plan), (xg, wg), dzg, create_graph=True)
    gx, gw, gdz = torch.autograd.grad(first, (xg, wg, dzg), (ex.to(dtype).cuda(), ew.to(dtype).cuda()))
    # d/dx <ew, G(x, dz)> = T(dz, ew); d/dw <ex, T(dz, w)> = G(ex, dz); d/d(dz) = F(ex, w) + F(x, ew)
    _, want_x, _ = ref.linear(*names, x, ew, index, dz)
    _, _, want_w = ref.linear(*names, ex, w, index, dz)
    want_z = ref.linear(*names, ex, w, index) + ref.linear(*names, x, ew, index)
    for got, want in ((gx, want_x), (gw, want_w), (gdz, want_z)):
        assert float((got.cpu().double() - want).abs().max() / want.abs().max()) < (1e-5 if dtype == F32 else 1e-12)


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_function_transforms():
    """torch.func and batched gradients over the op: the same as calls one by one."""
    names = "8x0e+4x1o", "6x0e+4x1o"
    x, w, _, index = inputs(*names, F64, 40, 3, 1)
    x, w, plan = x.cuda(), w.cuda(), groups_of(index, 3)
    lin, gen = oeq.GroupedLinear(*names), torch.Generator(device="cuda").manual_seed(2)
    loss = lambda p, q: lin(p, q, plan).square().sum()
    many = lambda t: torch.randn(5, *t.shape, device="cuda", generator=gen, dtype=F64)
    xs, ws = many(x), many(w)

    def one_by_one(p, q):
        p, q = p.clone().requires_grad_(True), q.clone().requires_grad_(True)
        return torch.autograd.grad(loss(p, q), (p, q))

    for got, want in zip(torch.func.grad(loss, (0, 1))(x, w), one_by_one(x, w)):
        assert torch.equal(got, want)
    assert torch.equal(torch.vmap(lambda p: lin(p, w, plan))(xs), torch.stack([lin(p, w, plan) for p in xs]))
    assert torch.equal(torch.vmap(lambda q: lin(x, q, plan))(ws), torch.stack([lin(x, q, plan) for q in ws]))
    want = [torch.stack(t) for t in zip(*[one_by_one(p, q) for p, q in zip(xs, ws)])]
    for got, t in zip(torch.vmap(torch.func.grad(loss, (0, 1)))(xs, ws), want):
        assert torch.equal(got, t)
    xg = xs.clone().requires_grad_(True)
    got, = torch.autograd.grad(torch.vmap(lambda p: lin(p, w, plan))(xg).square().sum(), xg)
    assert torch.equal(got, torch.stack([one_by_one(p, w)[0] for p in xs]))
    xg = x.clone().requires_grad_(True)
    z = lin(xg, w, plan)
    seeds = many(z)
    got, = torch.autograd.grad(z, xg, seeds, is_grads_batched=True, retain_graph=True)
    assert torch.equal(got, torch.stack([torch.autograd.grad(z, xg, e, retain_graph=True)[0] for e in seeds]))
    assert torch.func.jacrev(torch.func.grad(loss))(x, w).shape == (40, 20, 40, 20)


def test_weights_changed_in_place_are_noticed():
    x, w, dz, index = inputs("8x0e", "8x0e", F32, 50, 3, 1)
    plan, lin = groups_of(index, 3), oeq.GroupedLinear("8x0e", "8x0e")
    wg = w.float().cuda().requires_grad_(True)
    z = lin(x.float().cuda().requires_grad_(True), wg, plan)
    with torch.no_grad():
        wg.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        z.backward(dz.float().cuda())


def test_only_the_gradients_that_are_asked_for():
    x, w, dz, index = inputs("8x0e", "8x0e", F32, 50, 3, 1)
    plan, lin = groups_of(index, 3), oeq.GroupedLinear("8x0e", "8x0e")
    xg, wg, dzg = (t.float().cuda() for t in (x, w, dz))
    z = lin(xg.requires_grad_(True), wg, plan)
    z.backward(dzg)
    assert xg.grad is not None and wg.grad is None
    z = lin(xg.detach(), wg.requires_grad_(True), plan)
    z.backward(dzg)
    assert wg.grad is not None
    with torch.no_grad():
        assert not lin(xg, wg, plan).requires_grad


@pytest.mark.parametrize("dtype", [np.float32, np.float64], ids=["f32", "f64"])
def test_one_group_is_the_shared_tensor_product(dtype):
    """With one group the map is ``TensorProduct`` with shared dense weights and a second input of ones."""
    names, rows = ("32x0e+16x1o+8x2e", "24x0e+32x1o+8x2e"), 301
    problem = oeq.FullyConnectedTPProblem(names[0], "1x0e", names[1], irrep_dtype=dtype, weight_dtype=dtype)
    tp, lin = oeq.TensorProduct(problem, torch_op=True), oeq.GroupedLinear(*names)
    rng = np.random.default_rng(0)
    w = rng.normal(size=lin.weight_numel).astype(dtype)
    x = torch.from_numpy(rng.normal(size=(rows, problem.irreps_in1.dim)).astype(dtype)).cuda()
    ordered = np.zeros_like(w)
    tp.reorder_weights_e3nn_to_oeq(w, ordered, False)
    want = tp(x, x.new_ones(rows, 1), torch.from_numpy(ordered).cuda())
    got = lin(x, torch.from_numpy(w).cuda()[None], oeq.RowGroups(torch.zeros(rows, dtype=torch.int64, device="cuda"), 1))
    assert float((got - want).abs().max() / want.abs().max()) < (1e-5 if dtype == np.float32 else 1e-12)


# ------------------------------------------------------------------------------------------ a network's use of them

class Layer(torch.nn.Module):
    """Messages along edges, then a linear map with the weights of a node's element: the convolution and the map as a network
    runs them together."""

    def __init__(self, linear, conv, elements, numel):
        super().__init__()
        self.linear, self.conv = linear, conv
        self.w = torch.nn.Parameter(torch.randn(elements, numel, dtype=F64, generator=torch.Generator().manual_seed(2)))

    def forward(self, x, y, w_edge, edges, plan):
        return self.linear(self.conv(x, y, w_edge, *edges), self.w, plan)


def test_layer_of_a_convolution_and_a_grouped_map():
    """Energy, forces-like gradients that stay in the graph, and their derivatives, with the rows' groups built in the step."""
    from conftest import problem_by_name
    from helpers import conv_inputs, random_graph
    from oracle import tp_oracle as orc
    problem = problem_by_name("interaction_8", irrep_dtype=np.float64, weight_dtype=np.float64)
    names = str(problem.irreps_out), "8x0e+4x1o"
    nodes, elements = 60, 5
    rows, cols, _, perm = orc.coord_graph(*random_graph(nodes, 400, 1))
    x, y, w, _ = (torch.from_numpy(t) for t in conv_inputs(problem, nodes, 400, 2))
    species = torch.randint(0, elements, (nodes,), generator=torch.Generator().manual_seed(3))
    lin, conv = oeq.GroupedLinear(*names), oeq.TensorProductConv(problem, torch_op=True, deterministic=True)

    def step(layer, x, y, w, edges, plan):
        x = x.clone().requires_grad_(True)
        z = layer(x, y, w, edges, plan)
        force = torch.autograd.grad(z.square().sum(), x, create_graph=True)[0]
        return z, force, torch.autograd.grad(force.square().sum(), layer.w)[0]

    class Plain:
        def __call__(self, x, w, index):
            return ref.linear(*names, x, w, index)

    want = step(Layer(Plain(), lambda a, b, c, *e: orc.conv_torch(problem, a, b, c, *e), elements, lin.weight_numel), x, y, w,
                (torch.from_numpy(rows), torch.from_numpy(cols)), species)
    got = step(Layer(lin, conv.forward, elements, lin.weight_numel).cuda(), x.cuda(), y.cuda(), w.cuda(),
               tuple(torch.from_numpy(t).cuda() for t in (rows, cols, perm)), oeq.RowGroups(species.cuda(), elements))
    for g, t in zip(got, want):
        assert float((g.detach().cpu() - t.detach()).abs().max() / t.detach().abs().max()) < 1e-11


@pytest.mark.parametrize("dtype", TYPES, ids=TYPE_IDS)
def test_captured_and_replayed(dtype):
    """Groups, product and gradients in one CUDA graph, replayed on other groups and other values; an eager call of the
    same weights between."""
    names = "32x0e+16x1o", "48x0e+16x1o"
    lin, rows, groups = oeq.GroupedLinear(*names), 500, 6
    make = lambda seed: [t.to(dtype).cuda() if t.is_floating_point() else t.cuda() for t in inputs(*names, dtype, rows, groups, seed)]
    x, w, dz, index = make(0)

    def step():
        plan = oeq.RowGroups(index, groups)
        xg, wg = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        z = lin(xg, wg, plan)
        return (z.detach(), *torch.autograd.grad(z, (xg, wg), dz))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        for t, new in zip((x, w, dz, index), make(seed)):
            t.copy_(new)
        graph.replay()
        got = [t.clone() for t in out]
        for p, q in zip(got, step()):
            assert torch.equal(p, q)
    del graph
    gc.collect()


def test_two_streams():
    names = "64x0e+32x1o", "64x0e+32x1o"
    lin, sets = oeq.GroupedLinear(*names), []
    for seed, rows in ((1, 3001), (2, 2500)):
        x, w, dz, index = inputs(*names, F32, rows, 9, seed)
        sets.append([t.float().cuda() for t in (x, w, dz)] + [index.cuda()])

    def step(x, w, dz, index):
        plan = oeq.RowGroups(index, 9)
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        z = lin(x, w, plan)
        return (z.detach(), *torch.autograd.grad(z, (x, w), dz))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(*sets[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for run in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(run, want[k]))


def test_calls_from_several_threads_at_once():
    import threading
    names = "32x0e+16x1o+3x4e", "24x0e+16x1o+5x4e"
    data = []
    for seed, dtype in enumerate(TYPES * 2):
        x, w, dz, index = inputs(*names, dtype, 301, 5, seed)
        data.append([t.to(dtype).cuda() for t in (x, w, dz)] + [index.cuda()])

    def step(x, w, dz, index):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        z = oeq.GroupedLinear(*names)(x, w, oeq.RowGroups(index, 5))
        return (z.detach(), *torch.autograd.grad(z, (x, w), dz))

    want, got = [step(*d) for d in data], [None] * len(data)
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[k] = step(*data[k])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(data))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for run, expected in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(run, expected))


def test_more_than_2_to_the_31_values():
    """1.1 million rows of 2 048 values: offsets within the arrays pass 32 bits."""
    names, rows, groups = "128x0e+128x1o+128x2e+128x3o", 1_100_000, 3
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, 2048, device="cuda", generator=gen, dtype=BF16)
    lin = oeq.GroupedLinear(names, names)
    w = torch.randn(groups, lin.weight_numel, device="cuda", generator=gen, dtype=BF16)
    index = torch.arange(rows, device="cuda") % (groups + 1) - 1
    z = lin(x, w, oeq.RowGroups(index, groups))
    at = torch.cat([torch.arange(0, rows, 110_001), torch.arange(rows - 40, rows)])
    want = ref.linear(names, names, x[at.cuda()].cpu().double(), w.cpu().double(), index.cpu()[at])
    size = ref.linear(names, names, x[at.cuda()].cpu().double().abs(), w.cpu().double().abs(), index.cpu()[at])
    assert bool(((z[at.cuda()].cpu().double() - want).abs() <= ref.allowed(BF16, want, size, 128)).all())


def test_one_group_of_all_the_rows_there_can_be():
    """2^31 - 1 rows: the group's number of blocks, and a product that goes by the table of blocks (float64) and one that does not."""
    rows = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    plan = oeq.RowGroups.from_counts(torch.tensor([rows, 0], device="cuda"), rows)
    used = 2 ** 25
    assert plan.blocks.shape == (used + 1, 3) and plan.offsets.tolist() == [0, rows, rows]
    assert plan.blocks[-2:].tolist() == [[0, rows - 63, 63], [-1, 0, 0]]
    assert not plan.blocks[:used, 0].any() and bool((plan.blocks[:used - 1, 2] == 64).all())
    assert torch.equal(plan.blocks[:used, 1], torch.arange(0, rows, 64, dtype=torch.int32, device="cuda"))
    lin = oeq.GroupedLinear("1x0e", "1x0e")
    for dtype in (F64, BF16):
        x = torch.empty(rows, 1, dtype=dtype, device="cuda")
        for part in x.split(1 << 28):
            part.copy_((torch.arange(len(part), device="cuda") % 200)[:, None])
        z = lin(x, torch.tensor([[-2.0], [5.0]], dtype=dtype, device="cuda"), plan)
        assert all(torch.equal(p, q * -2) for p, q in zip(z.split(1 << 28), x.split(1 << 28)))
        del x, z, part
    del plan
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------ the ops

def test_ops():
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    lin = oeq.GroupedLinear("8x0e+4x1o", "6x0e+4x1o")
    x, w, dz, index = (t.cuda() for t in inputs("8x0e+4x1o", "6x0e+4x1o", F32, 40, 3, 1))
    x, w, dz = x.float(), w.float(), dz.float()
    plan = oeq.RowGroups(index, 3)
    ns = torch.ops.openequivariance_b200
    torch.library.opcheck(ns.row_groups.default, (index, 3), test_utils=checks)
    torch.library.opcheck(ns.row_groups_from_counts.default, (torch.tensor([20, 5, 9], device="cuda"), 40), test_utils=checks)
    for order in (plan.order, None):
        for kind, (a, b) in enumerate(((x, w), (dz, w), (x, dz))):
            args = (a.clone().requires_grad_(True), b, order, plan.offsets, plan.blocks, lin._number, kind)
            torch.library.opcheck(ns.grouped_linear.default, args, test_utils=checks)
    compiled = torch.compile(lambda p, q, i: lin(p, q, oeq.RowGroups(i, 3)), fullgraph=True)
    xg = x.clone().requires_grad_(True)
    z = compiled(xg, w, index)
    assert torch.equal(z.detach(), lin(x, w, plan))
    z.backward(dz)
    xe = x.clone().requires_grad_(True)
    lin(xe, w, plan).backward(dz)
    assert torch.equal(xg.grad, xe.grad)


def test_wrong_arguments_raise():
    lin = oeq.GroupedLinear("8x0e", "4x0e")
    cuda = lambda *shape, dtype=F32: torch.zeros(*shape, device="cuda", dtype=dtype)
    index = torch.zeros(10, dtype=torch.int64, device="cuda")
    plan = oeq.RowGroups(index, 3)
    for x, w, match in [(cuda(10, 7), cuda(3, 32), "rows must be"), (cuda(9, 8), cuda(3, 32), "rows must be"), (cuda(80), cuda(3, 32), "rows must be"),
                        (cuda(10, 8), cuda(2, 32), "weights must be"), (cuda(10, 8), cuda(3, 31), "weights must be"),
                        (cuda(10, 8), cuda(32), "weights must be"), (cuda(10, 8), cuda(3, 32, dtype=F64), "one type"),
                        (cuda(10, 8, dtype=torch.int32), cuda(3, 32, dtype=torch.int32), "must be float32")]:
        with pytest.raises(ValueError, match=match):
            lin(x, w, plan)
    for bad, groups in [(index.int(), 3), (index[None], 3), (index, 0), (index, -1), (index, 8192)]:
        with pytest.raises(ValueError):
            oeq.RowGroups(bad, groups)
    counts = torch.tensor([4, 6], device="cuda")
    for bad, rows in [(counts.int(), 10), (counts[None], 10), (counts, -1), (counts, 2 ** 31), (counts[:0], 10)]:
        with pytest.raises(ValueError):
            oeq.RowGroups.from_counts(bad, rows)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        with torch.autograd.forward_ad.dual_level():
            lin(torch.autograd.forward_ad.make_dual(cuda(10, 8), cuda(10, 8)), cuda(3, 32), plan)


def test_an_op_makes_the_map_that_it_names():
    """A map that no GroupedLinear of this process has, and names that are none."""
    names = "13x0e+3x1o", "11x0e+3x1o"
    x, w, dz, index = (t.cuda() for t in map_inputs(*names, 60, 4))
    plan = oeq.RowGroups(index, 4)
    op = torch.ops.openequivariance_b200.grouped_linear
    z = op(x, w, plan.order, plan.offsets, plan.blocks, "->".join(names), 0)
    assert torch.equal(z, oeq.GroupedLinear(*names)(x, w, plan))
    for bad, kind, match in (("13x0e", 0, "named by its irreps"), ("13x0e+3x1o->11x0e+3x1o", 3, "no such product"), ("12x0e->11x0e", 0, "rows must be")):
        with pytest.raises(ValueError, match=match):
            op(x, w, plan.order, plan.offsets, plan.blocks, bad, kind)
    with pytest.raises(RuntimeError, match="32 blocks"):
        op(x, w, plan.order, plan.offsets, plan.blocks, "+".join(["1x0e"] * 33) + "->1x0e", 0)


def map_inputs(irreps_in, irreps_out, rows, groups):
    gen = torch.Generator().manual_seed(7)
    a, b = Irreps(irreps_in), Irreps(irreps_out)
    numel = sum(m * n for m, p in a for n, q in b if p == q)
    return (torch.randn(rows, a.dim, generator=gen), torch.randn(groups, numel, generator=gen), torch.randn(rows, b.dim, generator=gen),
            torch.randint(0, groups, (rows,), generator=gen))


def test_an_exported_program_in_another_process(tmp_path):
    """The other process has made another map of the same widths before, with other weights in each place."""
    import subprocess
    import sys
    names, other = ("8x0e+8x0e", "4x0e+4x0e"), ("16x0e", "8x0e")
    x, w, _, index = (t.cuda() for t in map_inputs(*names, 50, 3))
    lin = oeq.GroupedLinear(*names)

    class Call(torch.nn.Module):
        def forward(self, x, w, index):
            return lin(x, w, oeq.RowGroups(index, 3))

    torch.export.save(torch.export.export(Call(), (x, w, index)), tmp_path / "call.pt2")
    torch.save((x.cpu(), w.cpu(), index.cpu()), tmp_path / "in.pt")
    code = f"""
import torch, openequivariance_b200 as oeq
oeq.GroupedLinear({other[0]!r}, {other[1]!r})
x, w, index = (t.cuda() for t in torch.load({str(tmp_path / 'in.pt')!r}))
torch.save(torch.export.load({str(tmp_path / 'call.pt2')!r}).module()(x, w, index).cpu(), {str(tmp_path / 'out.pt')!r})
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=ROOT)
    assert torch.equal(torch.load(tmp_path / "out.pt"), lin(x, w, oeq.RowGroups(index, 3)).cpu())


# ------------------------------------------------------------------------------------------ status

def test_the_check_waits_for_every_stream():
    """Streams of torch's pool do not block with the default stream: a copy of the status alone does not wait for them."""
    a, side, done = torch.randn(8192, 8192, device="cuda"), torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):                     # some 30 ms
            a @ a
        done.record()
    oeq.GroupedLinear.check_device_status()
    assert done.query()


def test_a_wait_that_runs_out_is_reported_once():
    from openequivariance_b200 import _native
    lib, side = _native.lib(), torch.cuda.Stream()
    assert lib.oeq_selftest_grouped_wait(2000, side.cuda_stream) == _native.OEQ_OK
    with pytest.raises(_native.OeqError, match="bounded wait"):
        oeq.GroupedLinear.check_device_status()
    oeq.GroupedLinear.check_device_status()
    assert lib.oeq_selftest_grouped_wait(0, side.cuda_stream) == _native.OEQ_ERR_INVALID
    check_linear("8x0e", "8x0e", F32, 70, 3)


@pytest.mark.parametrize("warp", [-1, 0, 3, 4, 7])
def test_a_warp_whose_wait_runs_out_comes_to_its_barriers(warp):
    """Three of the four warps that share a barrier go on; the kernel ends all the same."""
    from openequivariance_b200 import _native
    lib = _native.lib()
    assert lib.oeq_selftest_grouped_drain(warp, torch.cuda.current_stream().cuda_stream) == _native.OEQ_OK
    if warp < 0:
        oeq.GroupedLinear.check_device_status()
    else:
        with pytest.raises(_native.OeqError, match="bounded wait"):
            oeq.GroupedLinear.check_device_status()
    check_linear("8x0e", "8x0e", F32, 70, 3)


def test_products_on_their_way_are_over_before_a_kernel_gives_up():
    from openequivariance_b200 import _native
    assert _native.lib().oeq_selftest_grouped_issue(torch.cuda.current_stream().cuda_stream) == _native.OEQ_OK
    with pytest.raises(_native.OeqError, match="code 84"):
        oeq.GroupedLinear.check_device_status()
    check_linear("8x0e", "8x0e", F32, 70, 3)
