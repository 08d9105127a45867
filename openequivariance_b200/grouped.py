"""``RowGroups`` and ``GroupedLinear``: linear maps of irreps whose weights belong to groups of rows.

``TensorProduct`` with dense ("uvw") weights has one set for all rows or one for each row.  Equivariant networks also
keep one set for every *kind* of row -- a chemical element, a system of the batch, an expert chosen by a router -- and
multiply each row by the set of its group::

    groups = oeq.RowGroups(species, 89)                       # once per batch, on the GPU, no synchronisation
    linear = oeq.GroupedLinear("128x0e+128x1o", "128x0e+128x1o")
    z = linear(x, w, groups)                                  # x [rows, 512], w [89, linear.weight_numel]

The reference has no counterpart; its users index the weights by row (``w[species]``) or loop over the species.
"""

from __future__ import annotations

import functools

import torch

from . import _native
from .irreps import Irreps
from .tensor_product import _require_cuda


def _paths(irreps_in, irreps_out):
    """(input block, output block, slice of the weights, shape) of every pair of blocks with the same irrep."""
    paths, at = [], 0
    for i, (mul_in, ir_in) in enumerate(irreps_in):
        for o, (mul_out, ir_out) in enumerate(irreps_out):
            if ir_in == ir_out and mul_in * mul_out > 0:
                paths.append((i, o, slice(at, at + mul_in * mul_out), (mul_in, mul_out)))
                at += mul_in * mul_out
    return paths, at


@functools.lru_cache(maxsize=None)
def _widths(name):
    """Of the results of a map's product, its input gradient and its weight gradient."""
    irreps_in, irreps_out = (Irreps(part) for part in name.split("->"))
    return irreps_out.dim, irreps_in.dim, _paths(irreps_in, irreps_out)[1]


def _ops():
    _native.torch_lib()
    ns = torch.ops.openequivariance_b200
    blocks_of = lambda rows, groups: rows // 64 + min(rows, groups)

    @torch.library.register_fake("openequivariance_b200::row_groups")
    def _(index, groups):
        rows = index.shape[0]
        return (torch.empty_like(index), torch.empty_like(index), index.new_empty(groups + 1),
                index.new_empty((blocks_of(rows, groups), 3), dtype=torch.int32))

    @torch.library.register_fake("openequivariance_b200::row_groups_from_counts")
    def _(counts, rows):
        groups = counts.shape[0]
        return (counts.new_empty(rows), counts.new_empty(groups + 1),
                counts.new_empty((blocks_of(rows, groups), 3), dtype=torch.int32))

    @torch.library.register_fake("openequivariance_b200::grouped_linear")
    def _(a, b, order, offsets, blocks, map, kind):
        return a.new_empty(offsets.shape[0] - 1 if kind == 2 else a.shape[0], _widths(map)[kind])

    return ns.row_groups.default, ns.row_groups_from_counts.default, ns.grouped_linear.default


_row_groups, _row_groups_from_counts, _grouped_linear = _ops()     # (when the module is imported: a compiled call cannot load them)


class RowGroups:
    """The rows of a batch by their group: positions, offsets and a table of blocks, built on the GPU.

    ``index`` (int64, on the GPU) is the group of each row.  Rows whose group is not in ``0 .. num_groups - 1`` (padding)
    belong to none.

    * ``order``: the rows in the order of their groups, equal groups in the order of the rows, rows without a group last;
    * ``slots``: the position of each row in ``order``;
    * ``offsets``: position of the first row of each group, then the number of rows that have a group;
    * ``blocks``: int32 ``(group, first position, rows)`` of each run of 64 sorted rows of a group (its last run is
      shorter); unused entries, behind the others, are ``(-1, 0, 0)``.

    Sizes depend on the number of rows and groups alone: nothing waits for the GPU, and a construction can be captured
    into a CUDA graph.  At most 8191 groups.
    """

    def __init__(self, index: torch.Tensor, num_groups: int):
        _require_cuda(index)
        self.index, self.rows, self.num_groups = index, index.shape[0] if index.dim() else 0, int(num_groups)
        self.order, self.slots, self.offsets, self.blocks = _row_groups(index, self.num_groups)

    @classmethod
    def from_counts(cls, counts: torch.Tensor, rows: int) -> "RowGroups":
        """Groups of ``rows`` rows that lie in the order of their groups, from the number of rows of each (int64, on the
        GPU): the node counts of a batch of systems.  ``index`` is then the group of each row, -1 for rows behind the last
        group's; ``order`` and ``slots`` are None (every row is at its position).  Counts below zero are taken as zero,
        and groups are cut off at the last row."""
        _require_cuda(counts)
        self = cls.__new__(cls)
        self.rows, self.num_groups = int(rows), counts.shape[0] if counts.dim() else 0
        self.index, self.offsets, self.blocks = _row_groups_from_counts(counts, self.rows)
        self.order = self.slots = None
        return self


def _register(name):
    """Makes the map known, which refuses what cannot be made.  Maps are kept for the life of the process."""
    library = _native.torch_lib()
    code = library.oeq_torch_grouped_register(name.encode())
    if code < 0:
        raise RuntimeError(library.oeq_torch_grouped_error().decode(errors="replace"))
    _native.check(code)


class GroupedLinear:
    """``z[r] = x[r] W[group of r]`` for every irrep: the linear map of irreps with one set of weights per group of rows.

    A path joins every pair of input and output blocks with the same irrep::

        z[r, o, w, k] = sum over i, u of  W[g][i, o][u, w] x[r, i, u, k] / sqrt(number of (i, u) summed)

    ``weights`` is ``[groups, weight_numel]``: the paths with the input block outermost (``paths``: input block, output
    block, slice of the weights, shape), each row-major ``[channels of i, channels of o]`` -- e3nn's order, and the same
    normalisation as ``FullyConnectedTPProblem(irreps_in, "1x0e", irreps_out)``.  Rows without a group give zeros, and so
    do output blocks without a path.

    float32 (three TF32 products on the tensor cores; relative error below 1e-6, whatever the number of terms), bfloat16 and float16 (float32 sums,
    rounded once) and float64; the type is that of the tensors.  Derivatives of any order; gradients of weights are summed
    in a fixed order, so every result is the same in every run.  In float32 an infinity, a NaN or a number within 2^-12 of
    the largest one gives NaN in the results that it has a part in.

    The kernel is chosen for the map as a whole: with a path of l = 4 or above all of its paths run on FMA kernels in float32, bfloat16
    and float16 too, and with a multiplicity that is no multiple of 4 (16-bit types: 8) values are read one by one.

    An exported or pickled call holds the map's irreps and means the same map in every process that has imported this module.
    """

    def __init__(self, irreps_in, irreps_out):
        self.irreps_in, self.irreps_out = Irreps(irreps_in), Irreps(irreps_out)
        self.paths, self.weight_numel = _paths(self.irreps_in, self.irreps_out)
        self._map = f"{self.irreps_in}->{self.irreps_out}"      # the map as the op takes it: the same in every process
        _register(self._map)

    @property
    def _number(self):
        return self._map

    def forward(self, x: torch.Tensor, weights: torch.Tensor, groups: RowGroups) -> torch.Tensor:
        if not x.is_cuda or not weights.is_cuda:
            _require_cuda(x, weights)
        if x.dim() != 2 or x.shape[0] != groups.rows:
            raise ValueError(f"rows must be [{groups.rows}, {self.irreps_in.dim}], got {tuple(x.shape)}")
        return _grouped_linear(x, weights, groups.order, groups.offsets, groups.blocks, self._map, 0)

    __call__ = forward

    @staticmethod
    def check_device_status():
        """Raises if a kernel on the current device has abandoned a bounded wait since the last check.  Waits for all streams of
        the device."""
        _native.check(_native.lib().oeq_grouped_check())
