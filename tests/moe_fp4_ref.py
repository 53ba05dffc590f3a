"""Plain implementations, in 64 bits on the CPU, of the routing and 4-bit
operators: the definitions in include/megacu_b200.h, one statement at a time."""
from __future__ import annotations

import math

import torch

BLOCK = {0: 32, 1: 16}  # FP4_MX, FP4_NV
ELEMENTS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6],
                        dtype=torch.float64)
MX_SCALES = torch.tensor([2.0 ** (b - 127) for b in range(255)] + [math.nan],
                         dtype=torch.float64)
NV_SCALES = torch.tensor([m * 2.0 ** -9 for m in range(8)]
                         + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]
                         + [math.nan], dtype=torch.float64)
SCALES = {0: MX_SCALES, 1: NV_SCALES}


# ---- routing -------------------------------------------------------------------------

def sort(ids, experts, first, align, capacity):
    """(counts, offsets, row_of_slot, slot_of_row) by appending slot after slot."""
    lists = [[] for _ in range(experts)]
    for s, e in enumerate(ids.reshape(-1).tolist()):
        if 0 <= e - first < experts:
            lists[e - first].append(s)
    counts = [len(x) for x in lists]
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + -(-c // align) * align)
    row_of_slot, slot_of_row = [-1] * ids.numel(), [-1] * capacity
    for start, slots in zip(offsets, lists):
        for i, s in enumerate(slots):
            row_of_slot[s], slot_of_row[start + i] = start + i, s
    as_int = lambda x: torch.tensor(x, dtype=torch.int32)
    return (as_int(counts), as_int(offsets), as_int(row_of_slot).view(ids.shape),
            as_int(slot_of_row))


def dispatch(x, row_of_slot, rows):
    out = rows.clone()
    for t, row in enumerate(row_of_slot.tolist()):
        for r in row:
            if r >= 0:
                out[r] = x[t]
    return out


def combine(rows, weights, row_of_slot):
    """(sums, sums of magnitudes) in 64 bits."""
    tokens, topk = row_of_slot.shape
    w = torch.ones(tokens, topk, dtype=torch.float64) if weights is None else weights.double()
    y = torch.zeros(tokens, rows.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(y)
    for t, row in enumerate(row_of_slot.tolist()):
        for j, r in enumerate(row):
            if r >= 0:
                y[t] += w[t, j] * rows[r].double()
                mag[t] += (w[t, j] * rows[r].double()).abs()
    return y, mag


def combine_grad(dy, rows, weights, row_of_slot, drows):
    """(drows, dweights, sums of magnitudes of dweights) in 64 bits."""
    out = drows.double()
    dw = torch.zeros(row_of_slot.shape, dtype=torch.float64)
    mag = torch.zeros_like(dw)
    for t, row in enumerate(row_of_slot.tolist()):
        for j, r in enumerate(row):
            if r >= 0:
                out[r] = weights[t, j].double() * dy[t].double()
                prod = dy[t].double() * rows[r].double()
                dw[t, j], mag[t, j] = prod.sum(), prod.abs().sum()
    return out, dw, mag


# ---- 4-bit blocks --------------------------------------------------------------------

def quantize(x, fmt, g=1.0):
    """(codes [rows, cols], scale bytes [rows, blocks]) of g * x."""
    block = BLOCK[fmt]
    z = (x.double() * g).reshape(x.shape[0], -1, block)
    amax = z.abs().amax(-1)
    bad = ~torch.isfinite(z).all(-1)
    amax = torch.where(bad, torch.zeros_like(amax), amax)
    if fmt == 0:
        e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(-127, 127)
        byte = (e + 127).long()
    else:
        grid = NV_SCALES[:-1]
        v = (amax / 6).clamp(max=448)
        # 53 bits of quotient tell a 24-bit amax from six times any midpoint
        up = torch.searchsorted(grid, v.contiguous()).clamp(max=grid.numel() - 1)
        lo = (up - 1).clamp(min=0)
        dl, du = v - grid[lo], grid[up] - v
        byte = torch.where((dl < du) | ((dl == du) & (lo % 2 == 0)), lo, up)
        byte = torch.where(v == grid[up], up, byte)
    byte = torch.where(bad, torch.full_like(byte, 255 if fmt == 0 else 127), byte)
    s = SCALES[fmt][byte]
    a = z.abs()
    code = torch.zeros(z.shape, dtype=torch.int64)
    for border, tie_up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1),
                           (5.0, 0)):
        b = border * s[..., None]
        code += (a > b) | ((a == b) & bool(tie_up))
    code += 8 * torch.signbit(z)
    empty = bad | (s == 0)
    code = torch.where(empty[..., None], torch.zeros_like(code), code)
    return code.reshape(x.shape), byte


def pack(code, byte):
    """(data bytes [rows, cols / 2], tiled scale bytes)."""
    data = (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8)
    rows, nblk = byte.shape
    rt, kt = -(-rows // 128), -(-nblk // 4)
    tiled = torch.zeros(rt * kt * 512, dtype=torch.uint8)
    r, b = torch.meshgrid(torch.arange(rows), torch.arange(nblk), indexing="ij")
    tiled[scale_index(r, b, kt)] = byte.to(torch.uint8)
    return data, tiled


def scale_index(r, b, tiles_per_row):
    return ((r // 128) * tiles_per_row + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4


def values(data, tiled, fmt, g=1.0):
    """The values of a packed matrix in 64 bits."""
    d = data.long()
    rows, cols = d.shape[0], d.shape[1] * 2
    code = torch.stack((d & 15, d >> 4), -1).reshape(rows, cols)
    nblk = cols // BLOCK[fmt]
    r, b = torch.meshgrid(torch.arange(rows), torch.arange(nblk), indexing="ij")
    s = SCALES[fmt][tiled.long()[scale_index(r, b, -(-nblk // 4))]]
    return ELEMENTS[code] * s.repeat_interleave(BLOCK[fmt], 1) / g


def random_operand(gen, rows, cols, fmt, spread=3):
    """A quantised matrix of random codes and scales near 1."""
    code = torch.randint(0, 16, (rows, cols), generator=gen)
    nblk = cols // BLOCK[fmt]
    byte = (127 if fmt == 0 else 56) + torch.randint(-spread, spread + 1, (rows, nblk),
                                                     generator=gen)
    return pack(code, byte)


def product(a, b, alpha=1.0):
    """(alpha * a @ b^T, the same of magnitudes)."""
    return alpha * (a @ b.T), abs(alpha) * (a.abs() @ b.abs().T)


def swiglu(gate, up, gate_err=0.0, up_err=0.0):
    """(silu(g) * u, bound of its error for errors of g and u): |silu'| <= 1.1."""
    s = gate / (1 + torch.exp(-gate))
    err = 1.1 * gate_err * (up.abs() + up_err) + s.abs() * up_err
    return s * up, err
