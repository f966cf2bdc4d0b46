"""Paged cache on the GPU against the 64-bit oracle: writing, reading back, and the attention of new tokens.

Tolerances of the attention.  eps = half a step of the element type (bf16 2^-8, fp16 2^-11), u = 2^-24.  With A = sum of
softmax * |v| and Z = the largest sum of |q_d k_d| * scale of a row:
  * probabilities are rounded to the element type once: eps * A; the result is: eps * |out| <= eps * A;
  * scores are fp32 sums of D exact products, in the order of the matrix pipe: (D + 2) * u * Z each, which moves a
    weight by twice that (numerator and denominator), so 2 (D + 2) u Z * A; the long sums over N keys: 2 (N + 64) u * A, and exp2
    itself a few u: 16 u * A;
  * fp16 has a smallest step of 2^-24: half of it per probability and result, N * 2^-25 * max|v| + 2^-25.
The log-sum-exp is fp32 throughout: ((D + 2) Z + 2 (N + 64) + 16) * log2(e) * u, plus 2 u |lse|.
"""
import math

import pytest
import torch

from oracle import paged as O
from vqtree_amd.ops import paged_cache as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0**-24
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


class Cache:
    """A random cache on the CPU (pools, exponents, table, lengths) and its copy on the GPU."""

    WIDE = False  # whether the tables have room for 2^18 keys more

    def __init__(self, new, past, *, Hkv=2, G=1, D=128, page=16, dtype=torch.bfloat16, e4m3=False, seed=0, extra=0,
                 spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens = list(new), [a + b for a, b in zip(new, past)]
        self.Hkv, self.G, self.D, self.page, self.dtype, self.e4m3 = Hkv, G, D, page, dtype, e4m3
        need = [-(-n // page) for n in self.lens]
        n_pages = sum(need) + 2 + extra
        width = max(need + [1]) + 1 + (2**18 // page if Cache.WIDE else 0)
        order = torch.randperm(n_pages, generator=g).tolist()
        self.table = torch.full((len(new), width), -1, dtype=torch.int32)
        for s, n in enumerate(need):
            for c in range(n):
                self.table[s, c] = order.pop()
        self.free = order
        pools = []
        for k in range(2):
            x = torch.randn(n_pages, Hkv, page, D, generator=g) * (spread if k == 0 else 1.0)
            if e4m3:
                byte = torch.randint(118, 122, (n_pages, Hkv, page), generator=g, dtype=torch.int32)
                pools += [(x * 32).to(torch.float8_e4m3fn), byte.to(torch.uint8)]  # values around 2^5 * 2^-7
            else:
                pools += [x.to(dtype), None]
        self.k, self.k_exp, self.v, self.v_exp = pools
        T = sum(new)
        self.q = torch.randn(T, Hkv * G, D, generator=g).to(dtype)
        self.cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32)

    def exps(self, dev=None):
        if not self.e4m3:
            return {}
        return {"k_exp": self.k_exp.to(dev or "cpu"), "v_exp": self.v_exp.to(dev or "cpu")}

    def attend(self, q=None, **kw):
        q = self.q.to(DEV) if q is None else q
        return P.attn_paged(q, self.k.to(DEV), self.v.to(DEV), self.table.to(DEV), self.cu.to(DEV), self.kv_lens.to(DEV),
                            **self.exps(DEV), **kw)

    def want(self, **kw):
        return O.paged_attention(self.q, self.k, self.v, self.table, self.cu, self.kv_lens, **self.exps(), **kw)

    def check(self, causal=True, window=None, lse=True, softmax_scale=None, max_q_len=None):
        print("case", self.new, self.lens, self.Hkv, self.G, self.D, self.page, self.dtype, self.e4m3, causal, window, lse,
              max_q_len, flush=True)
        got = self.attend(causal=causal, window=window, return_lse=lse, softmax_scale=softmax_scale, max_q_len=max_q_len)
        torch.cuda.synchronize()
        compare(got if lse else (got, None), self.want(causal=causal, window=window, softmax_scale=softmax_scale), self)


def compare(got, want, c, rows=slice(None)):
    out, lse = got
    w_out, w_lse, A, Z = (x[rows] for x in want)
    eps = torch.finfo(c.dtype).eps / 2
    N, D = max(c.lens + [1]), c.D
    Z = Z[..., None]
    tol = (2 * eps + (2 * (D + 2) * Z + 2 * (N + 64) + 16) * U) * A
    if c.dtype == torch.float16:
        tol = tol + N * 2.0**-25 * float(c.v.float().abs().nan_to_num(0, 0, 0).max()) + 2.0**-25
    err = (out.double().cpu()[rows] - w_out).abs()
    assert torch.isfinite(err).all(), "non-finite output"
    assert (err <= tol).all(), f"out: {float((err / tol.clamp(min=1e-30)).max()):.3g} of the tolerance, max err {float(err.max()):.3g}"
    if lse is not None:
        lse = lse.double().cpu()[rows]
        same = lse == w_lse  # both -inf
        tol = ((D + 2) * Z[..., 0] + 2 * (N + 64) + 16) * 1.4427 * U + 2 * U * w_lse.abs()
        bad = ~(same | ((lse - w_lse).abs() <= tol))
        assert not bad.any(), f"lse: {int(bad.sum())} off, {float((lse - w_lse).abs().nan_to_num(0).max()):.3g}"


@pytest.fixture(params=["table", "wide_table"])
def table_width(request):
    """Which kernel a call takes and how it is cut up follows from the room in the tables, so a test that uses this runs for
    both: chunks of 65 rows and more with the few-rows kernel where the table ends behind the last page, and with their own."""
    Cache.WIDE = request.param == "wide_table"
    yield
    Cache.WIDE = False


both_widths = pytest.mark.usefixtures("table_width")

FORMS = [("bf16", False, 128, 1, 16), ("bf16", True, 128, 4, 64), ("f16", False, 64, 4, 32), ("f16", True, 64, 1, 16),
         ("bf16", False, 128, 8, 64), ("bf16", True, 64, 7, 128), ("f16", True, 128, 2, 256)]
LENGTHS = {
    "single": ([1, 1, 1], [0, 15, 300]),
    "long_single": ([1], [5000]),
    "few": ([5, 3, 1, 8], [60, 0, 64, 1000]),
    "chunk": ([150], [333]),
    "first_chunk": ([257], [0]),
    "mixed": ([70, 1, 0, 33, 1], [130, 640, 12, 0, 63]),
    "nothing": ([0, 0], [0, 77]),
}


@both_widths
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{'e4m3' if f[1] else '16'}-d{f[2]}-g{f[3]}-p{f[4]}")
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_attention(lengths, form):
    new, past = LENGTHS[lengths]
    dtype, e4m3, D, G, page = form
    c = Cache(new, past, Hkv=3 if G < 4 else 2, G=G, D=D, page=page, dtype=DTYPES[dtype], e4m3=e4m3, seed=len(lengths))
    if c.q.shape[0] == 0:
        out, lse = c.attend(return_lse=True)
        assert out.shape == c.q.shape and lse.shape == c.q.shape[:2]
        return
    c.check()
    c.check(lse=False, max_q_len=max(new))
    c.check(window=40)
    c.check(causal=False)


DEALS = {  # new, past, Hkv, G, D, page: how the work is dealt out (few-rows kernel / chunk kernel)
    "one_tile_many_parts": ([90], [3000], 2, 1, 128, 16),
    "tiles_in_equal_pieces": ([600], [4200], 2, 1, 64, 64),
    "line_of_tiles": ([70] * 5, [4300, 4200, 4100, 4000, 3900], 32, 1, 64, 128),
    "line_of_single_tokens": ([1] * 9, [5000, 10, 2500, 0, 7000, 300, 4000, 1999, 63], 4, 2, 64, 16),
    "more_than_64_sequences": ([1, 0, 2] * 50, list(range(0, 1500, 10)), 2, 4, 64, 32),
    "more_than_64_tiles": ([33, 70, 1] * 24, [i % 90 for i in range(72)], 1, 2, 64, 16),
    "long_tiles_beyond_64": ([70] * 66, [2100 + i for i in range(66)], 1, 1, 64, 256),
    "no_keys_at_all": ([100, 1], [0, 0], 2, 2, 64, 16),
    "whole_tiles_in_turns": ([600], [0], 128, 1, 64, 16),
    "many_short_tiles_of_32_rows": ([150, 3, 40], [0, 30, 64], 32, 2, 128, 16),
    "many_single_tokens": ([1] * 12, [7 * i * i for i in range(12)], 32, 1, 128, 16),
    "large_pages": ([65, 1], [5000, 4097], 2, 1, 64, 4096),
}


@both_widths
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("deal", DEALS, ids=str)
def test_ways_of_dealing_out(deal, e4m3):
    new, past, Hkv, G, D, page = DEALS[deal]
    c = Cache(new, past, Hkv=Hkv, G=G, D=D, page=page, e4m3=e4m3, seed=20, spread=2.0)
    if deal == "no_keys_at_all":
        c.kv_lens.zero_()
        c.lens = [0, 0]
        out, lse = c.attend(return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
        return
    want = c.want()
    for max_q in (None, max(new), 1):  # (the last hint is wrong where there are chunks: slower, not wrong)
        got = c.attend(return_lse=True, max_q_len=max_q)
        torch.cuda.synchronize()
        print(deal, e4m3, max_q, flush=True)
        compare(got, want, c)


@both_widths
@pytest.mark.parametrize("new", [[1], [80]])
def test_offsets_beyond_32_bits(new):
    """Pages that lie more than 4 GiB into the pools (and exponents far in): read, written and attended."""
    H, D, page, n_pages = 8, 128, 64, 36000
    c = Cache(new, [300], Hkv=H, D=D, page=page, seed=21)
    k, v = (torch.empty(n_pages, H, page, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    assert k.numel() * 2 > 2**32
    high = c.table.clone()
    for i in range(high.shape[1]):
        p = int(c.table[0, i])
        if p >= 0:
            high[0, i] = n_pages - 1 - p
            k[n_pages - 1 - p], v[n_pages - 1 - p] = c.k[p].to(DEV), c.v[p].to(DEV)
    out, lse = P.attn_paged(c.q.to(DEV), k, v, high.to(DEV), c.cu.to(DEV), c.kv_lens.to(DEV), return_lse=True)
    compare((out, lse), c.want(), c)
    rk, rv = P.paged_read(k, v, high.to(DEV), c.kv_lens.to(DEV), c.lens[0])
    assert torch.equal(rk[0].double().cpu(), O.rows_of(c.k, None, c.table[0], c.lens[0])[0])
    x = torch.randn(sum(new), H, D).to(torch.bfloat16)
    P.paged_write(x.to(DEV), x.to(DEV), k, v, high.to(DEV), c.cu.to(DEV), c.kv_lens.to(DEV))
    rk, rv = P.paged_read(k, v, high.to(DEV), c.kv_lens.to(DEV), c.lens[0])
    assert torch.equal(rv[0, :, 300:].cpu(), x.transpose(0, 1)) and torch.equal(rk[0, :, 300:].cpu(), x.transpose(0, 1))


@pytest.mark.parametrize("window", [0, 1, 63, 64, 129])
def test_windows(window):
    for e4m3 in (False, True):
        c = Cache([70, 3], [200, 500], D=64, page=16, G=2, e4m3=e4m3, seed=22)
        c.check(window=window)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window", [None, 0, 63, 129, 700])
def test_long_chunks(window, e4m3):
    c = Cache([1100, 2, 70], [300, 500, 0], Hkv=1, D=64, page=32, e4m3=e4m3, seed=24)
    c.check(window=window, max_q_len=1100)
    if window is None:
        c.check(causal=False)


@both_widths
@pytest.mark.parametrize("scale", [1e-6, 1.0, 30.0])
def test_scales(scale):
    """Flat, sharp and one-hot softmax: the tolerance is that of the scores the scale gives."""
    for new in ([1], [100]):
        c = Cache(new, [700], D=64, page=16, seed=23)
        got = c.attend(softmax_scale=scale, return_lse=True)
        compare(got, c.want(softmax_scale=scale), c)


# ---------------------------------------------------------------------------------------------------------------------
# writing and reading
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,page,H", [(128, 16, 3), (64, 64, 1)])
def test_write_then_read(dtype, e4m3, D, page, H):
    dt = DTYPES[dtype]
    new, past = [3, 0, 65, 1, 40], [14, 5, 0, 200, 63]
    c = Cache(new, past, Hkv=H, D=D, page=page, dtype=dt, e4m3=e4m3, seed=3)
    g = torch.Generator().manual_seed(4)
    T = sum(new)
    buf = torch.randn(T + 9, 3 * H * D, generator=g)  # columns of a projection; 9 rows behind the last sequence
    buf[:T] *= torch.logspace(-6, 3, T)[:, None]
    buf[2], buf[7, :D] = 0, 0
    buf[5, H * D + 3], buf[6, H * D + 5], buf[8, 2 * H * D + 1] = math.inf, -math.inf, math.nan
    buf[9, H * D] = 65504.0
    buf[10, :] *= 1e-6
    buf = buf.to(dt)
    k, v = buf[:, H * D:2 * H * D].view(-1, H, D), buf[:, 2 * H * D:].view(-1, H, D)
    gpu = [x.to(DEV) if x is not None else None for x in (c.k, c.v, c.k_exp, c.v_exp)]
    kg, vg = (x.view(-1, H, D) for x in buf.to(DEV)[:, H * D:].split(H * D, 1))
    assert not kg.is_contiguous()
    exps = dict(k_exp=gpu[2], v_exp=gpu[3]) if e4m3 else {}
    P.paged_write(kg, vg, gpu[0], gpu[1], c.table.to(DEV), c.cu.to(DEV), c.kv_lens.to(DEV), **exps)
    torch.cuda.synchronize()
    want = [c.k.clone(), c.v.clone(), None if c.k_exp is None else c.k_exp.clone(), None if c.v_exp is None else c.v_exp.clone()]
    for s, n in enumerate(new):
        for t in range(n):
            j = c.lens[s] - n + t
            p, o, row = int(c.table[s, j // page]), j % page, int(c.cu[s]) + t
            for pages, exp, x in ((want[0], want[2], k), (want[1], want[3], v)):
                if exp is None:
                    pages[p, :, o] = x[row]
                else:
                    values, byte = O.quantise_rows(x[row])
                    scaled = torch.ldexp(values, 127 - byte.int().unsqueeze(-1))
                    pages.view(torch.uint8)[p, :, o] = scaled.float().to(torch.float8_e4m3fn).view(torch.uint8)
                    exp[p, :, o] = byte
    bits = torch.uint8 if e4m3 else torch.int16
    for a, b in zip(gpu[:2], want[:2]):
        a, b = a.cpu().view(bits), b.view(bits)
        same = a == b
        if e4m3:  # a NaN keeps no sign
            same |= ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
        assert same.all(), f"{int((~same).sum())} elements differ"
    if e4m3:
        assert torch.equal(gpu[2].cpu(), want[2]) and torch.equal(gpu[3].cpu(), want[3])
    # and back
    n = max(c.lens) + 3
    rk, rv = P.paged_read(gpu[0], gpu[1], c.table.to(DEV), c.kv_lens.to(DEV), n, dtype=dt, **exps)
    for got, pages, exp in ((rk, want[0], want[2]), (rv, want[1], want[3])):
        for s in range(len(new)):
            x, _ = O.rows_of(pages, exp, c.table[s], c.lens[s])
            full = torch.zeros(H, n, D, dtype=torch.float64)
            full[:, :c.lens[s]] = x
            assert torch.equal(got[s].cpu().nan_to_num(7.0), full.to(dt).nan_to_num(7.0))
            assert torch.isfinite(full).sum() == torch.isfinite(got[s]).sum().cpu()


def test_every_e4m3_number_reads_back_exactly():
    """256 bit patterns under exponents 2^-126 .. 2^120, against the exact product rounded once."""
    page, D = 256, 64
    pages = torch.arange(256, dtype=torch.uint8).repeat(page * D // 256).view(1, 1, page, D)
    byte = torch.arange(256, dtype=torch.int32).clamp(1, 247).to(torch.uint8).view(1, 1, page)
    pages8 = pages.view(torch.float8_e4m3fn)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([page], dtype=torch.int32)
    exact = torch.ldexp(pages8.float().double(), byte.int().unsqueeze(-1) - 127)
    for dt in (torch.bfloat16, torch.float16):
        k, v = P.paged_read(pages8.to(DEV), pages8.to(DEV), table.to(DEV), lens.to(DEV), page, k_exp=byte.to(DEV),
                            v_exp=byte.to(DEV), dtype=dt)
        want = exact.to(dt)  # (torch rounds a double to 16 bits once)
        ok = exact.abs() <= torch.finfo(dt).max
        normal = ok & ((exact == 0) | (exact.abs() >= torch.finfo(dt).tiny))
        for got in (k.cpu(), v.cpu()):
            assert torch.equal(got[normal], want[normal])
            tiny = ok & ~normal  # results below the normal numbers: within a step of the smallest number, or flushed to it
            step = torch.finfo(dt).tiny * torch.finfo(dt).eps
            bound = torch.finfo(dt).tiny if dt == torch.bfloat16 else step
            assert ((got[tiny].double() - exact[tiny]).abs() <= bound).all()
            nan = torch.isnan(exact)
            assert torch.isnan(got[nan]).all()


def test_rows_that_have_no_place_are_skipped():
    """Behind the last sequence, before position 0, behind the table, on pages that are not there: nothing is written."""
    H, D, page = 2, 64, 16
    k = torch.randn(40, H, D, device=DEV).to(torch.bfloat16)
    pool = torch.zeros(4, H, page, D, dtype=torch.bfloat16, device=DEV)
    k_pages, v_pages = pool.clone(), pool.clone()
    table = torch.tensor([[1, 99], [-5, 2], [3, 3]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 20, 30, 33], dtype=torch.int32, device=DEV)
    lens = torch.tensor([20, 26, 34], dtype=torch.int32, device=DEV)  # the third has places 31, 32, 33: two behind the table
    P.paged_write(k, k, k_pages, v_pages, table, cu, lens)
    want = pool.clone()
    want[1] = k[:16].transpose(0, 1)       # sequence 0: positions 0 .. 15 on page 1, 16 .. 19 on no page
    want[2, :, :10] = k[20:30].transpose(0, 1)  # sequence 1: positions 16 .. 25
    want[3, :, 15] = k[30]
    assert torch.equal(k_pages, want) and torch.equal(v_pages, want)
    P.paged_write(k, k, k_pages, v_pages, table, cu, torch.tensor([-3, 4, 2], dtype=torch.int32, device=DEV))
    want[3, :, 0], want[3, :, 1] = k[31], k[32]  # sequence 1: no page; sequence 2: row 30 would be at position -1
    assert torch.equal(k_pages, want)


# ---------------------------------------------------------------------------------------------------------------------
# hidden places, missing pages, odd metadata
@both_widths
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,past", [([1, 1], [20, 333]), ([130], [70]), ([300, 5], [0, 900])])
def test_hidden_places_may_hold_anything(e4m3, new, past):
    """NaN and infinities in unused places of the last page, in keys above the causal limit and below the window, and on
    pages nobody reads."""
    c = Cache(new, past, D=128, page=64, e4m3=e4m3, seed=9)
    clean = c.want(window=50)
    bad = 0x7F if e4m3 else None
    for s, n in enumerate(c.lens):
        for j in range(0, (c.table.shape[1] - 1) * 64):
            p = int(c.table[s, j // 64])
            first = c.lens[s] - new[s] - 50  # the first row's window starts here
            if p >= 0 and (j >= n or j < first):
                for pool in (c.k, c.v):
                    if bad is None:
                        pool[p, :, j % 64] = math.nan if j % 2 else math.inf
                    else:
                        pool.view(torch.uint8)[p, :, j % 64] = bad
    for p in c.free:
        for pool in (c.k, c.v):
            pool.view(torch.uint8)[p] = 0x7F
    compare(c.attend(window=50, return_lse=True), clean, c)


@both_widths
@pytest.mark.parametrize("new", [7, 200])
def test_a_later_tokens_nan_does_not_reach_earlier_rows(new):
    c = Cache([new], [90], D=64, page=16, G=2, seed=2)
    clean = c.want()
    first = c.lens[0] - 3  # the last three tokens' values are poison
    for j in range(first, c.lens[0]):
        c.v[int(c.table[0, j // 16]), :, j % 16] = math.inf if j == first else math.nan
    out, lse = c.attend(return_lse=True)
    compare((out, lse), clean, c, rows=slice(0, new - 3))
    assert torch.isinf(out[new - 3]).all() and torch.isnan(out[new - 2:]).all()


@both_widths
def test_missing_pages_and_odd_lengths():
    c = Cache([1, 40, 3, 2], [300, 100, 0, 700], D=128, page=16, G=2, seed=5)
    c.table[0, 3], c.table[0, 18], c.table[1, 0], c.table[3, 1] = -1, c.k.shape[0], 2**31 - 1, -(2**31)
    c.table[2, :] = -1           # nothing there at all
    c.kv_lens[3] = 10_000        # more keys than the table has room for: the rows stand behind them all
    c.lens[3] = 10_000
    got = c.attend(return_lse=True)
    want = c.want()
    compare(got, want, c)
    assert (got[0][41:44] == 0).all() and torch.isinf(got[1][41:44]).all()
    got = c.attend(return_lse=True, window=20)
    compare(got, c.want(window=20), c)
    c.kv_lens[1], c.lens[1] = 25, 25  # fewer keys than new rows: the first 15 see nothing
    got = c.attend(return_lse=True)
    compare(got, c.want(), c)
    assert (got[0][1:16] == 0).all() and torch.isinf(got[1][1:16]).all()
    c.kv_lens[1], c.lens[1] = -7, 0
    compare(c.attend(return_lse=True), c.want(), c)


@both_widths
@pytest.mark.parametrize("new", [[1, 2], [90, 40]])
def test_rows_behind_the_last_sequence_are_left_alone(new):
    c = Cache(new, [100, 30], D=64, G=4, seed=6)
    T = sum(new)
    q = torch.cat([c.q, torch.full((37, 8, 64), math.nan, dtype=c.dtype)]).to(DEV)
    out = torch.full((T + 37, 8, 64), 5.0, dtype=c.dtype, device=DEV)
    got, lse = c.attend(q, out=out, return_lse=True)
    assert got is out and (out[T:] == 5).all()
    compare((out[:T], lse[:T]), c.want(), c)


@both_widths
def test_numbers_out_of_range_do_no_harm():
    """cu_q that decreases or runs past the rows: memory stays in bounds; rows of well-formed sequences come out right."""
    c = Cache([4, 40, 4], [50, 20, 30], D=64, seed=7)
    c.cu = torch.tensor([0, 4, 44, 2**31 - 1], dtype=torch.int32)
    out = c.attend()
    assert out.shape == c.q.shape and torch.isfinite(out.float()).all()
    c.cu = torch.tensor([0, -5, 2**31 - 1, -(2**31)], dtype=torch.int32)
    c.attend()
    torch.cuda.synchronize()
    # overlapping claims: a row goes to the first sequence that names it
    c.cu = torch.tensor([0, 44, 4, 48], dtype=torch.int32)
    got = c.attend(return_lse=True)
    c.cu = torch.tensor([0, 44, 44, 48], dtype=torch.int32)
    compare(got, c.want(), c)


# ---------------------------------------------------------------------------------------------------------------------
# layouts, streams, graphs, a whole run
@both_widths
@pytest.mark.parametrize("new", [[1, 1], [100, 3]])
def test_strided_tensors(new):
    """q as columns of a projection, out as rows of a wider buffer, key and value pages interleaved in one pool."""
    c = Cache(new, [200, 31], D=128, G=4, Hkv=2, page=32, seed=8)
    T = sum(new)
    kv = torch.stack([c.k, c.v], 1).to(DEV)  # [pages, 2, H, page, D]
    buf = torch.randn(T, 12, 128, device=DEV).to(c.dtype)
    buf[:, :8] = c.q.to(DEV)
    wide = torch.zeros(T, 16, 128, dtype=c.dtype, device=DEV)
    out, lse = P.attn_paged(buf[:, :8], kv[:, 0], kv[:, 1], c.table.to(DEV)[:, :-1], c.cu.to(DEV), c.kv_lens.to(DEV),
                            out=wide[:, 4:12], return_lse=True)
    compare((out, lse), c.want(), c)
    assert (wide[:, :4] == 0).all() and (wide[:, 12:] == 0).all()
    # a transposed query (last dimension not contiguous) is copied
    qt = c.q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    compare(P.attn_paged(qt, kv[:, 0], kv[:, 1], c.table.to(DEV), c.cu.to(DEV), c.kv_lens.to(DEV), return_lse=True), c.want(), c)


@both_widths
def test_another_stream_and_two_calls_at_once():
    a, b = Cache([1, 1], [3000, 700], seed=10, G=2), Cache([80], [900], seed=11, G=2, e4m3=True)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    gots = []
    args = [(c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), c.table.to(DEV), c.cu.to(DEV), c.kv_lens.to(DEV), c.exps(DEV)) for c in (a, b)]
    torch.cuda.synchronize()
    for stream, (*x, e) in zip((sa, sb), args):
        with torch.cuda.stream(stream):
            gots.append(P.attn_paged(*x, **e, return_lse=True))
    torch.cuda.synchronize()
    compare(gots[0], a.want(), a)
    compare(gots[1], b.want(), b)


@pytest.mark.parametrize("width", [64, 400, 2000])
@pytest.mark.parametrize("new", [[1, 1, 1], [130, 1, 20]])
def test_recorded_step_replays_on_new_lengths(new, width):
    """A whole step -- write, then attend -- recorded once: lengths, tables and rows change between the replays (and with
    the wide table the way the work is dealt out)."""
    H, G, D, page, S = 2, 2, 128, 16, 3
    T = sum(new)
    g = torch.Generator().manual_seed(12)
    pools = [torch.zeros(S * width, H, page, D, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2)]
    exps = [torch.ones(S * width, H, page, dtype=torch.uint8, device=DEV) for _ in range(2)]
    table = torch.randperm(S * width, generator=g).view(S, width).to(torch.int32).to(DEV)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    lens = torch.tensor(new, dtype=torch.int32, device=DEV)
    q, k, v = (torch.zeros(T, h, D, dtype=torch.bfloat16, device=DEV) for h in (H * G, H, H))
    e = dict(k_exp=exps[0], v_exp=exps[1])

    def step():
        P.paged_write(k, v, *pools, table, cu, lens, **e)
        return P.attn_paged(q, *pools, table, cu, lens, **e, return_lse=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        far = 100 if width == 64 else 2900
        lens.copy_(torch.tensor([n * (i + 1) + far * s * (i % 2) for s, n in enumerate(new)], dtype=torch.int32))
        graph.replay()
        got = out.clone(), lse.clone()
        again = step()  # (writes the same rows to the same places)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
        c = Cache([1], [1])
        c.lens, c.D, c.dtype = lens.tolist(), D, torch.bfloat16
        want = O.paged_attention(q.cpu(), pools[0].cpu(), pools[1].cpu(), table.cpu(), cu.cpu(), lens.cpu(),
                                 k_exp=exps[0].cpu(), v_exp=exps[1].cpu())
        compare(got, want, c)


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_run_of_steps(e4m3):
    """A prompt in three chunks, then single tokens, two sequences joining on the way: after every step the attention equals
    that over everything written so far, and the cache reads back as the tensors a dense operator takes."""
    from vqtree_amd.ops.attn_vq import attn_exact_decode

    H, G, D, page, width = 2, 2, 64, 16, 24
    g = torch.Generator().manual_seed(13)
    dt = torch.bfloat16
    pools = [torch.zeros(3 * width, H, page, D, dtype=torch.float8_e4m3fn if e4m3 else dt, device=DEV) for _ in range(2)]
    e = dict(zip(("k_exp", "v_exp"), (torch.ones(3 * width, H, page, dtype=torch.uint8, device=DEV) for _ in range(2)))) if e4m3 else {}
    table = torch.randperm(3 * width, generator=g).view(3, width).to(torch.int32).to(DEV)
    have = [0, 0, 0]
    for new in ([100, 0, 0], [61, 33, 0], [17, 1, 9], [1, 1, 1], [1, 1, 1], [4, 0, 2]):
        T = sum(new)
        q, k, v = (torch.randn(T, h, D, generator=g).to(dt).to(DEV) for h in (H * G, H, H))
        have = [a + b for a, b in zip(have, new)]
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        lens = torch.tensor(have, dtype=torch.int32, device=DEV)
        P.paged_write(k, v, *pools, table, cu, lens, **e)
        got = P.attn_paged(q, *pools, table, cu, lens, **e, return_lse=True)
        c = Cache([1], [1], dtype=dt, D=D)
        c.lens = have
        cpu = {n: x.cpu() for n, x in e.items()}
        compare(got, O.paged_attention(q.cpu(), pools[0].cpu(), pools[1].cpu(), table.cpu(), cu.cpu(), lens.cpu(), **cpu), c)
    # the last token of sequence 0, by the dense operator on the cache read back
    k, v = P.paged_read(*pools, table, lens, have[0], dtype=dt, **e)
    last = q[new[0] - 1].view(1, H * G, 1, D)
    dense = attn_exact_decode(last, k[:1].repeat_interleave(G, 1), v[:1].repeat_interleave(G, 1))
    assert (dense[0, :, 0].float() - got[0][new[0] - 1].float()).abs().max() <= 2.0**-6


# ---------------------------------------------------------------------------------------------------------------------
# new rows fewer than the buffer has room for
def poisoned_lse(rows, heads):
    """Leaves a block of NaN where the allocator takes the next [rows, heads] fp32 tensor from."""
    torch.full((rows, heads), math.nan, device=DEV)


@both_widths
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("n", [1, 5, 16, 40, 64, 65, 200])
def test_one_sequence_in_a_longer_buffer(n, G, e4m3):
    """The last chunk of a prompt fed through a buffer of fixed size: the sequence has the rows cu_q names, not the buffer's."""
    T, Hkv, D = 256, 2, 64
    c = Cache([n], [300], Hkv=Hkv, G=G, D=D, page=64, e4m3=e4m3, seed=30)
    want = c.want()
    q = torch.cat([c.q, torch.full((T - n, Hkv * G, D), math.nan, dtype=c.dtype)]).to(DEV)
    for max_q in (None, T, 10**9, n):
        out = torch.full((T, Hkv * G, D), 5.0, dtype=c.dtype, device=DEV)
        poisoned_lse(T, Hkv * G)
        got, lse = c.attend(q, out=out, return_lse=True, max_q_len=max_q)
        compare((got[:n], lse[:n]), want, c)
        assert (out[n:] == 5).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("width", [8, 1024])
@pytest.mark.parametrize("cuts", [
    ([0, 5], [0, 200], [0, 16], [0, 17], [0, 0], [0, 200], [0, 1]),
    ([0, 1, 33, 200], [0, 70, 71, 71], [0, 0, 16, 200], [0, 17, 34, 50], [0, 200, 200, 200], [0, 1, 2, 3]),
], ids=["one_sequence", "three_sequences"])
def test_recorded_attention_replays_on_other_chunks(cuts, width, e4m3):
    """Recorded once over a buffer of 200 rows, replayed on chunks of other lengths: sequences cross the 64 rows (16 tokens of
    4 heads) that part the two kernels in both directions."""
    T, H, G, D, page, S = 200, 2, 4, 64, 128, len(cuts[0]) - 1
    g = torch.Generator().manual_seed(31)
    c = Cache([1], [1], Hkv=H, G=G, D=D, page=page, e4m3=e4m3, seed=32, extra=S * 8)
    table = torch.full((S, width), -1, dtype=torch.int32)
    table[:, :8] = torch.randperm(c.k.shape[0], generator=g)[:S * 8].view(S, 8)
    q = torch.randn(T, H * G, D, generator=g).to(c.dtype)
    cu, lens = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (S + 1, S))
    out = torch.zeros(T, H * G, D, dtype=c.dtype, device=DEV)
    args = (q.to(DEV), c.k.to(DEV), c.v.to(DEV), table.to(DEV), cu, lens)
    exps = c.exps(DEV)

    def step():
        return P.attn_paged(*args, **exps, return_lse=True, out=out)[1]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lse = step()
    for i, cut in enumerate(cuts):
        print("cut", cut, flush=True)
        new = [b - a for a, b in zip(cut, cut[1:])]
        c.lens = [n + 50 + 211 * s + 97 * i for s, n in enumerate(new)]
        cu.copy_(torch.tensor(cut, dtype=torch.int32))
        lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
        out.fill_(5.0), lse.fill_(math.nan)
        graph.replay()
        n = cut[-1]
        want = O.paged_attention(q[:n], c.k, c.v, table, torch.tensor(cut), torch.tensor(c.lens), **c.exps())
        compare((out[:n], lse[:n]), want, c)
        assert (out[n:] == 5).all()
        replayed = out.clone()
        out.fill_(5.0)
        step()
        assert torch.equal(replayed, out)


@both_widths
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [[1, 2], [90, 3]])
def test_lengths_up_to_the_largest_int(new, e4m3):
    """More keys than any table has room for: the rows stand behind them all and, without a window, see them all; with one they
    see what it leaves of them."""
    c = Cache(new, [300, 30], D=64, page=128, G=2, e4m3=e4m3, seed=33)
    for length in (2**30 + 500, 2**31 - 1):
        c.kv_lens[0] = length
        kept, c.lens = c.lens, [512, c.lens[1]]  # (the sums run over the keys the table holds)
        got = c.attend(return_lse=True)
        whole = c.want()
        compare(got, whole, c)
        compare(c.attend(return_lse=True, causal=False), c.want(causal=False), c)
        n = new[0]
        for window in (2**31 - 2, length - 200, 100):
            out, lse = c.attend(return_lse=True, window=window)
            compare((out, lse), c.want(window=window), c)
            if window == 100:
                assert (out[:n] == 0).all() and (lse[:n] == -math.inf).all()
        c.lens = kept


@both_widths
@pytest.mark.parametrize("new", [[1], [20], [90]])
def test_exponent_byte_0_counts_as_1(new):
    """In every kernel and for keys and values alike: byte 0, which the write never leaves, is 2^-126 as byte 1 is."""
    c = Cache(new, [200], D=64, page=16, G=2, e4m3=True, seed=34)
    got = []
    for low in (0, 1):
        c.k_exp[:], c.v_exp[:] = 118, 1
        c.v_exp[:, :, ::3], c.k_exp[:, :, 1::5] = low, low
        out, lse = c.attend(return_lse=True)
        k, v = P.paged_read(c.k.to(DEV), c.v.to(DEV), c.table.to(DEV), c.kv_lens.to(DEV), c.lens[0], dtype=c.dtype, **c.exps(DEV))
        got.append((out, lse, k, v))
    assert (got[0][0] != 0).any() and torch.isfinite(got[0][0]).all()
    for a, b in zip(*got):
        assert torch.equal(a, b)


@both_widths
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,past,Hkv,G", [
    ([1, 3], [400, 70], 1, 40), ([9], [300], 1, 130), ([1], [200], 1, 600), ([2, 1], [500, 33], 300, 1), ([66], [200], 300, 1),
    ([1] * 300, [(37 * i) % 500 for i in range(300)], 1, 2), ([5, 0, 20] * 90, [(53 * i) % 300 for i in range(270)], 2, 4),
], ids=["g40", "g130", "g600", "300_heads", "300_heads_chunk", "300_sequences", "270_sequences"])
def test_many_heads_and_many_sequences(new, past, Hkv, G, e4m3):
    """Groups of heads larger than a tile, more key heads than compute units, more sequences than a few waves hold."""
    c = Cache(new, past, Hkv=Hkv, G=G, D=64, page=32, e4m3=e4m3, seed=35)
    got = c.attend(return_lse=True)
    compare(got, c.want(), c)


@both_widths
@pytest.mark.parametrize("new", [[1, 4], [90, 1]])
def test_states_of_two_caches_merge(new):
    """Attention over the first keys and over the rest, joined by merge_state_in_place, is attention over all of them.  Each of
    the two states is within compare()'s tolerance of its part, the parts' weights add up to one, and the result is rounded once
    more: 3 roundings instead of 2 (eps * A each); the weights follow the log-sum-exps, whose errors move a weight by ln 2 times
    that, twice."""
    from vqtree_amd.ops.triton_fused_vq_attn import merge_state_in_place

    c = Cache(new, [300, 150], D=128, page=16, G=2, seed=36)
    cut = 6  # pages; the second sequence's rows stand behind them too
    args = (c.q.to(DEV), c.k.to(DEV), c.v.to(DEV))
    cu = c.cu.to(DEV)
    first = torch.full((2,), cut * 16, dtype=torch.int32, device=DEV)
    a, sa = P.attn_paged(*args, c.table[:, :cut].to(DEV), cu, first, causal=False, return_lse=True)
    b, sb = P.attn_paged(*args, c.table[:, cut:].contiguous().to(DEV), cu, c.kv_lens.to(DEV) - cut * 16, return_lse=True)
    merge_state_in_place(a, sa, b, sb)
    w_out, w_lse, A, Z = c.want()
    eps, N = torch.finfo(c.dtype).eps / 2, max(c.lens)
    lse_tol = ((c.D + 2) * Z + 2 * (N + 64) + 16) * 1.4427 * U + 8 * U * w_lse.abs()
    tol = (3 * eps + (2 * (c.D + 2) * Z[..., None] + 2 * (N + 64) + 16) * U + 2 * 0.6932 * lse_tol[..., None]) * A
    assert ((a.double().cpu() - w_out).abs() <= tol).all()
    assert ((sa.double().cpu() - w_lse).abs() <= lse_tol).all()
