"""Paged cache and the attention over it in 64 bits, sequence by sequence (test infrastructure)."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def quantise_rows(x):
    """(values [.., D] float64, byte [..] uint8): rows as the 8-bit cache holds them, from the definition -- the nearest
    multiple of the spacing of e4m3 numbers (2^-3 of the power of two below, 2^-9 below 2^-6), ties to even, of x / 2^e with e
    the smallest integer that brings the row's largest magnitude to 448 or less."""
    top = 1.875 * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    x = x.double().clamp(-top, top)
    values, bytes_ = torch.empty_like(x), torch.empty(x.shape[:-1], dtype=torch.uint8)
    for at, row in zip(torch.cartesian_prod(*(torch.arange(n) for n in x.shape[:-1])).reshape(-1, x.dim() - 1).tolist(),
                       x.reshape(-1, x.shape[-1])):
        most = max([abs(float(v)) for v in row if not math.isnan(float(v))] + [0.0])
        e = -126
        while e < 120 and most > 448.0 * 2.0**e:
            e += 1
        y = row / 2.0**e
        size = torch.frexp(y.abs())[1] - 1  # y in [2^size, 2^(size + 1))
        step = torch.pow(2.0, (size.clamp(min=-6) - 3).double())
        values[tuple(at)] = torch.round(y / step) * step * 2.0**e
        bytes_[tuple(at)] = e + 127
    return values, bytes_


def rows_of(pages, exps, table_row, n):
    """[H, n, D] float64 and [n] bool (the row's page is there): the first n rows of one sequence."""
    P, H, page, D = pages.shape
    out, there = torch.zeros(H, n, D, dtype=torch.float64), torch.zeros(n, dtype=torch.bool)
    for j in range(0, n, page):
        m = min(page, n - j)
        p = int(table_row[j // page])
        if 0 <= p < P:
            x = pages[p, :, :m].double() if exps is None else pages[p, :, :m].float().double()
            if exps is not None:
                x = x * torch.ldexp(torch.ones((), dtype=torch.float64), exps[p, :, :m].int() - 127).unsqueeze(-1)
            out[:, j:j + m], there[j:j + m] = x, True
    return out, there


def paged_attention(q, k_pages, v_pages, block_table, cu_q, kv_lens, *, k_exp=None, v_exp=None, softmax_scale=None,
                    causal=True, window=None):
    """(out [T,Hq,D], lse [T,Hq] base 2, weight_v [T,Hq,D], score_size [T,Hq]) in 64 bits.  weight_v = sum of softmax * |v|
    and score_size = the largest sum of |q_d k_d| * scale of a visible key are what rounding errors are relative to.  Rows
    behind the last sequence are NaN.  Hidden keys take no part, whatever they hold."""
    T, Hq, D = q.shape
    Hkv, page = k_pages.shape[1], k_pages.shape[2]
    scale = softmax_scale or 1.0 / math.sqrt(D)
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64)
    weight_v, size = torch.zeros_like(out), torch.zeros_like(lse)
    cap = block_table.shape[1] * page
    for s in range(block_table.shape[0]):
        a, b, n_keys = int(cu_q[s]), int(cu_q[s + 1]), int(kv_lens[s])
        held = max(0, min(n_keys, cap))
        k, there = rows_of(k_pages, k_exp, block_table[s], held)
        v, _ = rows_of(v_pages, v_exp, block_table[s], held)
        j = torch.arange(held)
        for t in range(a, b):
            i = n_keys - (b - a) + (t - a)
            seen = there.clone()
            if causal:
                seen &= j <= i
                if window is not None:
                    seen &= i - j <= window
            if not seen.any():
                out[t], lse[t] = 0.0, -math.inf
                continue
            ks = k[:, seen].repeat_interleave(Hq // Hkv, 0)
            vs = v[:, seen].repeat_interleave(Hq // Hkv, 0)
            qt = q[t].double()
            z = torch.einsum("hd,hjd->hj", qt, ks) * scale
            l = torch.logsumexp(z, -1)
            p = torch.exp(z - l[:, None])
            out[t] = torch.einsum("hj,hjd->hd", p, vs)
            weight_v[t] = torch.einsum("hj,hjd->hd", p, vs.abs())
            size[t] = (torch.einsum("hd,hjd->hj", qt.abs(), ks.abs()) * scale).amax(-1)
            lse[t] = l / math.log(2.0)
    return out, lse, weight_v, size
