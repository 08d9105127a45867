"""Grouped linear maps without a GPU: paths, refusals, and the C ABI's checks (none of these calls reaches a device)."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import openequivariance_b200 as oeq
from openequivariance_b200 import _native
import grouped_reference as ref
from conftest import ROOT


def test_paths_and_weights():
    lin = oeq.GroupedLinear("8x0e+3x1o+2x0e", "4x0e+5x1e+6x0e+1x1o")
    assert lin.paths == [(0, 0, slice(0, 32), (8, 4)), (0, 2, slice(32, 80), (8, 6)), (1, 3, slice(80, 83), (3, 1)),
                         (2, 0, slice(83, 91), (2, 4)), (2, 2, slice(91, 103), (2, 6))]
    assert lin.weight_numel == 103
    assert oeq.GroupedLinear("2x1o", "3x1e").weight_numel == 0


def test_reference_is_the_fully_connected_product():
    """The map of one group, and its normalisation, against the oracle of the shared dense product with a second input of 1."""
    from oracle import tp_oracle as orc
    problem = oeq.FullyConnectedTPProblem("5x0e+3x1o+2x0e", "1x0e", "4x0e+6x1o", irrep_dtype=np.float64, weight_dtype=np.float64)
    rng = np.random.default_rng(0)
    x, w = rng.normal(size=(7, problem.irreps_in1.dim)), rng.normal(size=problem.weight_numel)
    want = orc.tp_forward(problem, x, np.ones((7, 1)), w)
    got = ref.linear("5x0e+3x1o+2x0e", "4x0e+6x1o", torch.from_numpy(x), torch.from_numpy(w)[None], torch.zeros(7, dtype=torch.int64))
    np.testing.assert_allclose(got.numpy(), want, rtol=1e-13, atol=1e-13)


def test_maps_are_registered_once():
    numbers = []
    threads = [threading.Thread(target=lambda: numbers.append(oeq.GroupedLinear("9x0e+1x2e", "7x0e+2x2e")._number)) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(numbers)) == 1


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oeq.RowGroups(torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oeq.RowGroups.from_counts(torch.ones(3, dtype=torch.int64), 3)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oeq.GroupedLinear("2x0e", "2x0e")(torch.zeros(3, 2), torch.zeros(1, 4), None)


def test_too_many_blocks_are_refused():
    with pytest.raises(_native.OeqError, match="32 blocks"):
        oeq.GroupedLinear("+".join(["1x0e"] * 33), "1x0e")
    with pytest.raises(_native.OeqError, match="64 paths"):
        oeq.GroupedLinear("+".join(["1x0e"] * 9), "+".join(["1x0e"] * 8))
    with pytest.raises(_native.OeqError, match="2\\^30 weights"):
        oeq.GroupedLinear("40000x0e", "40000x0e")


def test_abi_refuses_bad_arguments():
    lib = _native.lib()
    handle = C.c_void_p()
    irrep = (_native._Irrep * 1)(_native._Irrep(4, 1, 1))
    assert lib.oeq_grouped_create(None, 1, irrep, 1, C.byref(handle)) == _native.OEQ_ERR_INVALID
    assert lib.oeq_grouped_create(irrep, 1, irrep, 1, None) == _native.OEQ_ERR_INVALID
    bad = (_native._Irrep * 1)(_native._Irrep(4, 1, 3))
    assert lib.oeq_grouped_create(bad, 1, irrep, 1, C.byref(handle)) == _native.OEQ_ERR_INVALID and not handle.value
    assert lib.oeq_grouped_create(irrep, 1, irrep, 1, C.byref(handle)) == _native.OEQ_OK
    assert lib.oeq_grouped_weight_numel(handle) == 16 and lib.oeq_grouped_weight_numel(None) == 0
    null = [None] * 6
    assert lib.oeq_grouped_forward(None, 0, 5, 2, *null, None) == _native.OEQ_ERR_INVALID
    assert lib.oeq_grouped_forward(handle, 4, 5, 2, *null, None) == _native.OEQ_ERR_INVALID       # dtype
    assert lib.oeq_grouped_forward(handle, 0, -1, 2, *null, None) == _native.OEQ_ERR_INVALID
    assert lib.oeq_grouped_forward(handle, 0, 2 ** 31, 2, *null, None) == _native.OEQ_ERR_INVALID
    assert lib.oeq_grouped_forward(handle, 0, 5, 0, *null, None) == _native.OEQ_ERR_INVALID
    assert lib.oeq_grouped_forward(handle, 0, 5, 8192, *null, None) == _native.OEQ_ERR_INVALID
    assert lib.oeq_grouped_forward(handle, 0, 5, 2, *null, None) == _native.OEQ_ERR_INVALID       # null arrays
    assert lib.oeq_grouped_backward_weights(handle, 0, 5, 2, *[None] * 5, None, 0, None) == _native.OEQ_ERR_INVALID
    assert b"null" in lib.oeq_last_error()
    assert lib.oeq_grouped_forward(handle, 0, 0, 2, *null, None) == _native.OEQ_OK               # no rows: nothing to do
    assert lib.oeq_row_groups(5, 2, *[None] * 5, None, 0, None) == _native.OEQ_ERR_INVALID
    assert lib.oeq_row_groups_from_counts(5, 0, *[None] * 4, None) == _native.OEQ_ERR_INVALID
    assert lib.oeq_grouped_destroy(handle) == _native.OEQ_OK


@pytest.mark.parametrize("rows,groups", [(0, 1), (1, 1), (1, 8191), (8192, 10), (8193, 10), (100000, 8191), (2 ** 31 - 1, 8191)])
def test_sizes(rows, groups):
    """The table holds the blocks of every division of the rows: as many groups as there are rows, each with one row more than
    whole blocks."""
    lib = _native.lib()
    blocks, used = lib.oeq_row_groups_blocks(rows, groups), min(rows, groups)
    whole = (rows - used) // 64
    assert blocks >= whole + used and blocks == rows // 64 + used
    assert lib.oeq_row_groups_workspace_bytes(rows, groups) <= 1200 * (groups + 1) * 4


def test_reference_of_row_groups():
    order, slots, offsets, blocks = ref.row_groups([2, 0, -1, 2, 5, 0], 3)
    assert order.tolist() == [1, 5, 0, 3, 2, 4] and slots.tolist() == [2, 0, 4, 3, 5, 1]
    assert offsets.tolist() == [0, 2, 2, 4] and blocks.tolist() == [[0, 0, 2], [2, 2, 2], [-1, 0, 0]]
    index, offsets, _ = ref.from_counts([2, -1, 9], 5)
    assert index.tolist() == [0, 0, 2, 2, 2] and offsets.tolist() == [0, 2, 2, 5]


def test_selftests_refuse_bad_arguments():
    lib = _native.lib()
    for warp in (-2, 8):
        assert lib.oeq_selftest_grouped_drain(warp, None) == _native.OEQ_ERR_INVALID
    for polls in (0, 2 ** 20 + 1):
        assert lib.oeq_selftest_grouped_wait(polls, None) == _native.OEQ_ERR_INVALID


@pytest.mark.parametrize("offset", [4, 8, 16])
def test_abi_refuses_a_workspace_that_is_not_aligned(offset):
    """Partial sums are read 32 bytes at a time: an address between faults on the device, so the call ends before a launch."""
    lib, handle = _native.lib(), C.c_void_p()
    irrep = (_native._Irrep * 1)(_native._Irrep(4, 1, 1))
    assert lib.oeq_grouped_create(irrep, 1, irrep, 1, C.byref(handle)) == _native.OEQ_OK
    some = C.c_void_p(1 << 20)
    assert lib.oeq_grouped_backward_weights(handle, 1, 5, 2, some, some, None, some, some, C.c_void_p((1 << 20) + offset), 1 << 30, None) == _native.OEQ_ERR_INVALID
    assert b"aligned to 32 bytes" in lib.oeq_last_error()
    assert lib.oeq_grouped_destroy(handle) == _native.OEQ_OK


def test_a_map_is_the_same_in_every_process():
    """What a traced graph holds names the map, whichever maps a process has made before.  The two maps agree in all widths and lay their
    weights out differently."""
    import subprocess
    import sys
    code = "import sys, openequivariance_b200 as oeq; print([oeq.GroupedLinear(*m.split('/'))._number for m in sys.argv[1:]])"
    maps = ["8x0e+8x0e/4x0e+4x0e", "16x0e/8x0e"]
    run = lambda names: eval(subprocess.run([sys.executable, "-c", code, *names], capture_output=True, text=True, check=True, cwd=ROOT).stdout)
    first, second = run(maps), run(maps[::-1])
    assert first == second[::-1] and first[0] != first[1]


def test_a_traced_call_holds_the_irreps():
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    lin = oeq.GroupedLinear("8x0e+4x1o", "6x0e+4x1o")
    with FakeTensorMode():
        x, w, index = torch.empty(10, 20, device="cuda"), torch.empty(3, 64, device="cuda"), torch.zeros(10, dtype=torch.int64, device="cuda")
        graph = make_fx(lambda x, w, index: lin(x, w, oeq.RowGroups(index, 3)))(x, w, index).graph
    calls = [n for n in graph.nodes if "grouped_linear" in str(n.target)]
    assert len(calls) == 1 and "8x0e+4x1o->6x0e+4x1o" in calls[0].args


def test_pickled():
    import pickle
    lin = pickle.loads(pickle.dumps(oeq.GroupedLinear("3x0e", "5x0e+1x1o")))
    assert lin._map == "3x0e->5x0e+1x1o" and lin.weight_numel == 15


def test_maps_that_are_no_maps_are_refused():
    from openequivariance_b200 import grouped
    for name in ("3x0e", "3x0e->3", "3x0e->3x", "3x0e->3x0", "3x0e->3x0x", "3x0e+->3x0e", "-1x0e->1x0e", "1x0e->1x0e ", "9999999999x0e->1x0e", "a->b"):
        with pytest.raises(RuntimeError, match="named by its irreps"):
            grouped._register(name)
    grouped._register("->")
    grouped._register("12x0e->")
