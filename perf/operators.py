"""Workloads of the products whose weights belong to groups of rows, as programs that use them run them.

A network keeps one set of dense weights for every kind of row: a chemical element, a system of the batch, an expert that a
router picked.  A batch comes with the group of each row (or with the number of rows of each group, when the rows already
lie in order), and every layer then multiplies a row by the weights of its group.

  op         index      row groups from the group of each row: positions, offsets and the table of blocks
             counts     the same from the number of rows of each group
             forward    row groups and the product
             gradients  row groups, the product and the gradients of rows and weights: a training step
  irreps_in, irreps_out    of the rows; a path joins every pair of blocks with the same irrep
  dtype      f32 | f64 | bf16 | f16
  rows, groups
  by         index | counts: how the batch comes to its groups
  skew       groups have shares in proportion to rank ** -skew
  without    share of the rows that belong to no group (padding): their results are zero
"""

import functools
import itertools
import math

import torch

own = False

BLOCK = 64      # rows of an entry of the block table
DTYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}

NEQUIP = "32x0e+32x1o+32x2e"
FC = "64x0e+64x1o+64x2e"
MACE = "128x0e+128x1o+128x2e"
MACE_LARGE = "128x0e+128x1o+128x2e+128x3o"


def listed():
    def groups(name, op, rows, groups, skew=0.0, without=0.0):
        return {"name": name, "op": op, "rows": rows, "groups": groups, "skew": skew, "without": without}

    def linear(name, op, irreps_in, irreps_out, dtype, rows, groups, by="index", skew=0.0, without=0.0):
        return {"name": name, "op": op, "irreps_in": irreps_in, "irreps_out": irreps_out, "dtype": dtype, "rows": rows,
                "groups": groups, "by": by, "skew": skew, "without": without}

    return [
        # the elements of one molecule: what a call costs when there is almost nothing to sort
        groups("groups_molecule", "index", 27, 10),
        # the elements of a very large structure, some rows of padding
        groups("groups_index_1m", "index", 1_000_000, 89, 1.0, 0.05),
        # the node counts of a batch of small structures
        groups("groups_counts_50k", "counts", 50_000, 1000, 0.3, 0.02),
        # energy and forces of one small molecule
        linear("linear_molecule_f32", "gradients", MACE, MACE, "f32", 27, 10),
        # a training batch of structures of many elements, a few of them common
        linear("linear_mace_5k_f32", "gradients", MACE, MACE, "f32", 4999, 89, skew=1.5),
        # the wide model on a large structure
        linear("linear_mace_large_50k_f32", "gradients", MACE_LARGE, MACE_LARGE, "f32", 50_000, 10, skew=0.5),
        # inference of a narrow model, three elements
        linear("linear_nequip_20k_f32", "forward", NEQUIP, NEQUIP, "f32", 20_000, 3),
        # potentials are trained in double precision where energies have to be conserved
        linear("linear_fc64_10k_f64", "gradients", FC, FC, "f64", 10_007, 8, skew=1.0),
        # scalar features through experts, a training step in half precision
        linear("linear_scalars_64k_bf16", "gradients", "512x0e", "1024x0e", "bf16", 65_536, 64, skew=0.3),
        # inference with one set of weights for each system of the batch
        linear("linear_systems_100k_bf16", "forward", MACE, MACE, "bf16", 100_000, 256, by="counts", skew=0.3),
        # a gated block: multiplicities that fit no tile, two blocks of one irrep, an irrep that comes to nothing, padding
        linear("linear_odd_3k_f32", "gradients", "33x0e+17x1o+5x2e+3x2o", "19x0e+40x0e+21x1o+6x2e", "f32", 3001, 7,
               skew=0.7, without=0.1),
        # a handful of rows, each of its own group: the weights are what is read
        linear("linear_rows_8_f16", "forward", "256x0e+256x1o", "256x0e+256x1o", "f16", 8, 16),
    ]


def draw(rng):
    def spread(least, most):
        return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))

    op = rng.choice(("index", "counts", "forward", "forward", "gradients", "gradients", "gradients"))
    skew, without = round(rng.choice((0.0, rng.uniform(0.1, 1.8))), 2), rng.choice((0.0, 0.0, round(rng.uniform(0.01, 0.3), 2)))
    if op in ("index", "counts"):
        return {"op": op, "rows": spread(1, 1_000_000), "groups": spread(1, 2000), "skew": skew, "without": without}
    dtype = rng.choice(("f32", "f32", "f32", "bf16", "bf16", "f16", "f64"))
    width = {"f64": 64, "f32": 256}.get(dtype, 512)
    lmax = rng.randrange(4)
    same = rng.random() < 0.5
    mul = spread(3, width) if rng.random() < 0.4 else 2 ** rng.randint(3, int(math.log2(width)))
    other = mul if same else spread(3, width)
    name = lambda m: "+".join("%dx%d%s" % (m, l, "eo"[l % 2]) for l in range(lmax + 1))  # noqa: E731
    d = (lmax + 1) ** 2
    # no more values in a batch, and no more multiply-adds, than the largest listed case has
    most = min(100_000, 50_000 * 2048 // (d * max(mul, other)), 50_000 * 128 * 2048 // (d * mul * other))
    if dtype == "f64":
        most //= 8
    groups = spread(1, min(512, 200_000_000 // ((lmax + 1) * mul * other)))
    return {"op": op, "irreps_in": name(mul), "irreps_out": name(other), "dtype": dtype, "rows": spread(1, most),
            "groups": groups, "by": rng.choice(("index", "index", "counts")), "skew": skew, "without": without}


# ------------------------------------------------------------------------------------------ what a program has in hand

def blocks_of(irreps):
    """(multiplicity, irrep, components, first column) of each block."""
    out, at = [], 0
    for term in irreps.replace(" ", "").split("+"):
        mul, ir = term.split("x")
        out.append((int(mul), ir, 2 * int(ir[:-1]) + 1, at))
        at += int(mul) * (2 * int(ir[:-1]) + 1)
    return out


def dim_of(irreps):
    return sum(m * d for m, _, d, _ in blocks_of(irreps))


@functools.lru_cache(maxsize=None)
def paths_of(irreps_in, irreps_out):
    """(input block, output block, first weight, factor): every pair of blocks with the same irrep; an output's
    products are divided by the square root of the number of its input channels."""
    a, b = blocks_of(irreps_in), blocks_of(irreps_out)
    fan = {ir: sum(m for m, other, _, _ in a if other == ir) for _, ir, _, _ in a}
    out, at = [], 0
    for i, o in itertools.product(range(len(a)), range(len(b))):
        if a[i][1] == b[o][1]:
            out.append((i, o, at, 1.0 / math.sqrt(fan[a[i][1]])))
            at += a[i][0] * b[o][0]
    return out


def weight_numel(irreps_in, irreps_out):
    a, b = blocks_of(irreps_in), blocks_of(irreps_out)
    return sum(a[i][0] * b[o][0] for i, o, _, _ in paths_of(irreps_in, irreps_out))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, groups = case["rows"], case["groups"]
    share = torch.arange(1, groups + 1, device="cuda", dtype=torch.float64) ** -case["skew"]
    bounds = (share / share.sum()).cumsum(0)[:-1].contiguous()
    index = torch.searchsorted(bounds, torch.rand(rows, device="cuda", dtype=torch.float64, generator=gen), right=True)
    if case["without"]:
        index[torch.rand(rows, device="cuda", generator=gen) < case["without"]] = -1
    state = {"op": case["op"], "rows": rows, "groups": groups, "index": index, "counts": None}
    if case.get("by", case["op"]) == "counts":
        state["index"], state["counts"] = None, torch.bincount(index[index >= 0], minlength=groups)
    if "irreps_in" in case:
        def normal(*shape):
            return torch.randn(*shape, device="cuda", generator=gen).to(DTYPES[case["dtype"]])

        state.update(irreps=(case["irreps_in"], case["irreps_out"]), x=normal(rows, dim_of(case["irreps_in"])),
                     w=normal(groups, weight_numel(case["irreps_in"], case["irreps_out"])))
        if case["op"] == "gradients":
            state["dz"] = normal(rows, dim_of(case["irreps_out"]))
            state["x"].requires_grad_(True)
            state["w"].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------ one pass

@functools.lru_cache(maxsize=None)
def _linear(irreps_in, irreps_out):
    """A network makes its operators once."""
    import openequivariance_b200 as oeq
    return oeq.GroupedLinear(irreps_in, irreps_out)


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def _run_own(state):
    import openequivariance_b200 as oeq
    if state["counts"] is None:
        groups = oeq.RowGroups(state["index"], state["groups"])
    else:
        groups = oeq.RowGroups.from_counts(state["counts"], state["rows"])
    if state["op"] == "index":
        return groups.order, groups.slots, groups.offsets, groups.blocks
    if state["op"] == "counts":
        return groups.index, groups.offsets, groups.blocks
    linear = _linear(*state["irreps"])
    if state["op"] == "forward":
        with torch.no_grad():
            return linear(state["x"], state["w"], groups)
    z = linear(state["x"], state["w"], groups)
    return (z.detach(), *torch.autograd.grad(z, (state["x"], state["w"]), state["dz"]))


def _table(counts, rows):
    """Offsets of the groups among the sorted rows, and the table of blocks (group, first position, rows): whole
    blocks of a group, then its rest; unused entries are (-1, 0, 0)."""
    groups = counts.shape[0]
    ends = counts.cumsum(0).clamp(max=rows)
    offsets = torch.cat([ends.new_zeros(1), ends])
    each = (offsets.diff() + BLOCK - 1) // BLOCK
    last = each.cumsum(0)
    b = torch.arange(rows // BLOCK + min(rows, groups), device=counts.device)
    used = b < last[-1]
    g = torch.searchsorted(last, b, right=True).clamp(max=groups - 1)
    first = offsets[g] + (b - (last - each)[g]) * BLOCK
    table = torch.stack([g, first, (offsets[g + 1] - first).clamp(max=BLOCK)], dim=1)
    return offsets, torch.where(used[:, None], table, table.new_tensor([-1, 0, 0])).to(torch.int32)


def _groups(state):
    """order, slots, index, offsets, blocks."""
    rows, groups = state["rows"], state["groups"]
    place = torch.arange(rows, device="cuda")
    if state["counts"] is not None:
        offsets, blocks = _table(state["counts"], rows)
        index = torch.searchsorted(offsets[1:].contiguous(), place, right=True)
        return place, place, torch.where(index < groups, index, -1), offsets, blocks
    index = state["index"]
    key = torch.where((index >= 0) & (index < groups), index, groups)
    order = torch.sort(key, stable=True).indices
    slots = torch.empty_like(order).scatter_(0, order, place)
    offsets, blocks = _table(torch.bincount(key, minlength=groups + 1)[:groups], rows)
    return order, slots, index, offsets, blocks


def _run_plain(state):
    order, slots, index, offsets, blocks = _groups(state)
    if state["op"] == "index":
        return order, slots, offsets, blocks
    if state["op"] == "counts":
        return index, offsets, blocks
    # rows of a block of the table side by side, short blocks filled with zeros: one batched product for each path
    x, w, dz = state["x"].detach(), state["w"].detach(), state.get("dz")
    dtype, wide = x.dtype, torch.float64 if x.dtype == torch.float64 else torch.float32
    group, first, rows_of = blocks.long().unbind(1)
    place = torch.arange(BLOCK, device=x.device)
    real = place < rows_of[:, None]
    source = torch.where(real, order[(first[:, None] + place).clamp(max=x.shape[0] - 1)], x.shape[0])   # last: no row
    group = group.clamp(min=0)
    a, b = (blocks_of(r) for r in state["irreps"])
    paths = paths_of(*state["irreps"])
    pad = lambda t: torch.cat([t.to(wide), t.new_zeros(1, t.shape[1], dtype=wide)])[source]     # [blocks, BLOCK, dim]

    def take(t, block):             # [blocks, BLOCK * components, channels]
        m, _, d, at = block
        return t[:, :, at:at + m * d].unflatten(2, (m, d)).transpose(2, 3).flatten(1, 2)

    def give(parts, layout):        # [blocks, BLOCK * components, channels] of each block (None: zeros) -> rows
        out = torch.zeros(x.shape[0] + 1, sum(m * d for m, _, d, _ in layout), device=x.device, dtype=wide)
        flat = [(torch.zeros(len(group), BLOCK * d, m, device=x.device, dtype=wide) if p is None else p)
                .unflatten(1, (BLOCK, d)).transpose(2, 3).flatten(2) for p, (m, _, d, _) in zip(parts, layout)]
        out[source] = torch.cat(flat, dim=2)
        return out[:-1].to(dtype)

    def total(parts):
        return functools.reduce(torch.add, parts) if parts else None

    weights = [w[:, at:at + a[i][0] * b[o][0]].unflatten(1, (a[i][0], b[o][0])).to(wide)[group] for i, o, at, _ in paths]
    xs = pad(x)
    z = give([total([take(xs, a[i]) @ m * f for (i, o, _, f), m in zip(paths, weights) if o == n]) for n in range(len(b))], b)
    if state["op"] == "forward":
        return z
    gz = pad(dz)
    dx = give([total([take(gz, b[o]) @ m.transpose(1, 2) * f for (i, o, _, f), m in zip(paths, weights) if i == n])
               for n in range(len(a))], a)
    dw = [torch.zeros(w.shape[0], a[i][0], b[o][0], device=w.device, dtype=wide)
          .index_add_(0, group, take(xs, a[i]).transpose(1, 2) @ take(gz, b[o]) * f).flatten(1) for i, o, _, f in paths]
    return z, dx, torch.cat(dw, dim=1).to(dtype)


# ------------------------------------------------------------------------------------------ what a pass must do

def work(case):
    """Bytes: a call reads its inputs and writes its outputs once; the gradients read the output's gradient once for
    both.  Operations: one product a path forward, two backward."""
    rows, groups = case["rows"], case["groups"]
    blocks = rows // BLOCK + min(rows, groups)
    plan = 8 * (groups + 1) + 12 * blocks + 8 * rows
    plan += 8 * groups if case.get("by", case["op"]) == "counts" else 16 * rows
    if "irreps_in" not in case:
        return {"bytes": plan, "flops": 0}
    a, b = blocks_of(case["irreps_in"]), blocks_of(case["irreps_out"])
    paths = paths_of(case["irreps_in"], case["irreps_out"])
    s = {"f32": 4, "f64": 8}.get(case["dtype"], 2)
    used = int(round(rows * (1.0 - case["without"])))
    weights = min(used, groups) * weight_numel(case["irreps_in"], case["irreps_out"])      # of the groups with rows
    x, z = dim_of(case["irreps_in"]), dim_of(case["irreps_out"])
    flops = sum(2.0 * used * a[i][0] * b[o][0] * a[i][2] for i, o, _, _ in paths)
    total = plan + (used * x + weights + rows * z) * s
    if case["op"] == "gradients":
        total += (used * (x + z) + weights + rows * x + groups * weight_numel(case["irreps_in"], case["irreps_out"])) * s
        flops *= 3
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    """From the definition, a group at a time: z_r = x_r W_g / sqrt(n) for every irrep of every row r of group g."""
    state = prepare(case, seed)
    rows, groups = case["rows"], case["groups"]
    if "irreps_in" not in case:
        return None
    if state["counts"] is None:
        member = state["index"].tolist()
        rows_of = [[] for _ in range(groups)]
        for r, g in enumerate(member):
            if g >= 0:
                rows_of[g].append(r)
    else:
        at = 0
        rows_of = []
        for n in state["counts"].tolist():
            rows_of.append(list(range(at, at + n)))
            at += n
    a, b = blocks_of(case["irreps_in"]), blocks_of(case["irreps_out"])
    x, w = state["x"].detach().double(), state["w"].detach()
    z = torch.zeros(rows, dim_of(case["irreps_out"]), dtype=torch.float64, device="cuda")
    gradients = case["op"] == "gradients"
    if gradients:
        dz, dx = state["dz"].double(), torch.zeros_like(x)
        dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    for g, members in enumerate(rows_of):
        if not members:
            continue
        r = torch.tensor(members, device="cuda")
        begin = 0
        for mul_i, ir_i, d, col_i in a:
            fan = sum(m for m, ir, _, _ in a if ir == ir_i)
            for mul_o, ir_o, _, col_o in b:
                if ir_i != ir_o:
                    continue
                end = begin + mul_i * mul_o
                matrix = w[g, begin:end].double().reshape(mul_i, mul_o) / math.sqrt(fan)
                left = x[r, col_i:col_i + mul_i * d].reshape(-1, mul_i, d)
                z[r, col_o:col_o + mul_o * d] += torch.einsum("ruk,uw->rwk", left, matrix).flatten(1)
                if gradients:
                    right = dz[r, col_o:col_o + mul_o * d].reshape(-1, mul_o, d)
                    dx[r, col_i:col_i + mul_i * d] += torch.einsum("rwk,uw->ruk", right, matrix).flatten(1)
                    dw[g, begin:end] = torch.einsum("ruk,rwk->uw", left, right).flatten() / math.sqrt(fan)
                begin = end
    return (z, dx, dw) if gradients else z
