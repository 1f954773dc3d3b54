"""e4m3 numbers and their blocks from the definitions, in 64 bits on the host."""
import torch

F64, E4M3 = torch.float64, torch.float8_e4m3fn
BLOCK, PAGE = 128, 64


def power(largest):
    """The smallest power of two s >= 2^-100 with largest <= 448 s, tried from below."""
    largest = torch.as_tensor(largest, dtype=F64)
    p = torch.full_like(largest, 2.0 ** -100)
    for _ in range(240):
        p = torch.where(largest > 448.0 * p, 2.0 * p, p)
    return p


def nearest(v):
    """The nearest number of e4m3 (ties to even): steps of 2^-9 up to 2^-6, an eighth of the power of two below from there on; NaN for what is not finite."""
    v = v.to(F64)
    size = torch.where(torch.isfinite(v), v.abs(), 0.0).clamp_min(2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    return torch.where(torch.isfinite(v), torch.round(v / step) * step, float("nan"))


def finite_size(x):
    return torch.where(torch.isfinite(x), x.abs(), 0.0).to(F64)


def blocks(x, rows):
    """(values of the codes [n, k], scales [k blocks, row blocks]) of a matrix."""
    n, k = x.shape
    groups, row_blocks = -(-k // BLOCK), -(-n // rows)
    size = torch.zeros(row_blocks * rows, groups * BLOCK, dtype=F64)
    size[:n, :k] = finite_size(x)
    s = power(size.view(row_blocks, rows, groups, BLOCK).amax((1, 3)))
    wide = s.repeat_interleave(rows, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return nearest(x.to(F64) / wide), s.t().contiguous()


def same(a, b):
    """Equal numbers, NaN where NaN is."""
    a, b = a.to(F64), b.to(F64)
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def write(codes, scales, rows, table, seq_slots, cu, lens):
    """The blocks (values of codes [pages, heads, 64, dim], scales [pages, heads], both 64 bits) after the new rows, page by page."""
    codes, scales = codes.clone(), scales.clone()
    for b, length in enumerate(lens):
        at = length - (cu[b + 1] - cu[b])
        while at < length:
            first, end, page = at % PAGE, min(length - at // PAGE * PAGE, PAGE), int(table[seq_slots[b], at // PAGE])
            token = cu[b + 1] - length + at
            x = rows[token:token + end - first].to(F64).transpose(0, 1)
            s = power(finite_size(x).amax((1, 2)))
            if first:
                s = torch.maximum(s, scales[page])
                codes[page, :, :first] = nearest(codes[page, :, :first] * (scales[page] / s)[:, None, None])
            codes[page, :, first:end] = nearest(x / s[:, None, None])
            scales[page] = s
            at += end - first
    return codes, scales
