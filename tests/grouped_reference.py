"""Row groups and grouped linear maps written out in 64 bits on the CPU, and what a kernel's result may differ by."""
import numpy as np
import torch

from openequivariance_b200 import Irreps

BLOCK = 64


def table(counts, rows):
    """offsets and the table of blocks of groups with these numbers of rows (already within the rows)."""
    offsets, blocks, at = [0], [], 0
    for g, n in enumerate(counts):
        blocks += [(g, at + b, min(BLOCK, n - b)) for b in range(0, n, BLOCK)]
        at += n
        offsets.append(at)
    blocks += [(-1, 0, 0)] * (rows // BLOCK + min(rows, len(counts)) - len(blocks))
    return np.array(offsets, dtype=np.int64), np.array(blocks, dtype=np.int32).reshape(-1, 3)


def row_groups(index, groups):
    """order, slots, offsets, blocks."""
    index = np.asarray(index)
    key = np.where((index >= 0) & (index < groups), index, groups)
    order = np.argsort(key, kind="stable")
    slots = np.empty_like(order)
    slots[order] = np.arange(len(order))
    return (order, slots, *table(np.bincount(key, minlength=groups + 1)[:groups].tolist(), len(index)))


def from_counts(counts, rows):
    """index, offsets, blocks."""
    taken, left = [], rows
    for n in counts:
        taken.append(min(max(int(n), 0), left))
        left -= taken[-1]
    index = np.repeat(np.arange(len(taken) + 1), taken + [left])
    index[index == len(taken)] = -1
    return (index, *table(taken, rows))


def linear(irreps_in, irreps_out, x, w, index, dz=None):
    """z and, with dz, (z, dx, dw) of float64 tensors; the same of the absolute values bounds the rounding errors."""
    a, b = Irreps(irreps_in), Irreps(irreps_out)
    z = x.new_zeros(x.shape[0], b.dim)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for g in range(w.shape[0]):
        r = torch.nonzero(index == g).flatten()
        if not len(r):
            continue
        at = 0
        for (mul_i, ir_i), s_i in zip(a, a.slices()):
            fan = sum(m for m, ir in a if ir == ir_i)
            for (mul_o, ir_o), s_o in zip(b, b.slices()):
                if ir_i != ir_o or mul_i * mul_o == 0:
                    continue
                c = fan ** -0.5
                m = w[g, at:at + mul_i * mul_o].reshape(mul_i, mul_o)
                left = x[r][:, s_i].reshape(len(r), mul_i, ir_i.dim)
                z[r, s_o] += c * torch.einsum("ruk,uw->rwk", left, m).flatten(1)
                if dz is not None:
                    right = dz[r][:, s_o].reshape(len(r), mul_o, ir_i.dim)
                    dx[r, s_i] += c * torch.einsum("rwk,uw->ruk", right, m).flatten(1)
                    dw[g, at:at + mul_i * mul_o] = c * torch.einsum("ruk,rwk->uw", left, right).flatten()
                at += mul_i * mul_o
    return z if dz is None else (z, dx, dw)


def allowed(dtype, want, size, terms):
    """Largest difference of a result from `want`: `size` is the sum of the products' absolute values, `terms` their number.

    Every type: half a step of the result's own rounding (and of the smallest number of float16), and one step of the sum's
    type for each addition: the tensor cores' sums are cut off, not rounded, and an input to an FMA chain is rounded
    once more by the scale.  float32 products are made of TF32 parts, x = hi + lo with |lo| <= 2^-11 |x|: without lo.lo
    (2^-22), and with lo cut to 11 bits in either factor (2^-21 each).
    """
    half = torch.finfo(dtype).eps / 2
    step = 2.0 ** -52 if dtype == torch.float64 else 2.0 ** -23
    split = 2.0 ** -22 + 2 * 2.0 ** -21 if dtype == torch.float32 else 0.0
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return half * want.abs() + ((terms + 4) * step + split) * size + least


def allowed_norm(chain, chains):
    """Largest |result - exact| / |exact| (Frobenius norms) of float32 sums on the tensor cores of random values, sums being ended after
    `chain` additions and `chains` of them added up.

    An addition to an accumulator cuts off up to a step of the sum, 2^-23, towards zero: half of it on average, and as all of them go one
    way a chain is short by chain / 2 steps at most (its running sums are no larger on average than its end).  The sum of the chains is short by
    the same share.  Additions of chains round to nearest, half a step each in no direction: the root of their number.  Products: without
    lo.lo (2^-22), lo cut to 11 bits in either factor (2^-21 each), the scale on a factor and its two parts' sum half a step each.
    """
    return chain / 2 * 2.0 ** -23 + 2.0 ** -22 + 2 * 2.0 ** -21 + chains ** 0.5 * 2.0 ** -24 + 2 * 2.0 ** -24


def allowed_norm_rounded(chain, chains):
    """The same of sums that round to nearest: half a step of the running sum for each addition, in no direction, the running sums' squares
    being half of the end's on average; then the sum of the chains in the same way, and the scale and the result."""
    return ((chain / 2) ** 0.5 + (chains / 2) ** 0.5 + 2) * 2.0 ** -24
