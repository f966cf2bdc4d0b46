"""What is measured of the paged key / value cache: writing new tokens into it (with 8-bit storage on the way), reading
it back as plain tensors, and the attention of new tokens over it, from single tokens to long chunks.

The cache is two pools of pages, [pages, kv_heads, page, dim].  In 16 bits a row is stored as it is; in 8 bits it is
stored as e4m3 values next to one power-of-two exponent per row (a byte: value = e4m3 * 2^(byte - 127)).  A sequence's
rows are found through its row of the block table.  With `own` false every operator runs in its plain form, torch
operations in 32 bits; with `own` true the same inputs go to the framework's entry points.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
LOG2E = 1.4426950408889634


def _case(name, op, new, past, *, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", store="same", window=-1,
          causal=True, lse=False):
    return {"name": name, "op": op, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "store": store, "window": window, "causal": causal, "lse": lse}


def _texts(values):
    return ",".join(str(int(v)) for v in values)


def listed():
    spread = lambda n, lo, hi, step: _texts(lo + (i * step) % (hi - lo) for i in range(n))  # noqa: E731
    return [
        # one generation step of 64 conversations: a row per head and sequence; latency
        _case("write_step_e4m3", "write", _texts([1] * 64), spread(64, 90, 4000, 613), store="e4m3"),
        # a prompt of 8192 tokens of a 32-head model enters the cache
        _case("write_prompt_e4m3", "write", "8192", "0", kv_heads=32, store="e4m3", page=64),
        # continuous batching: chunks of unequal prompts and single tokens together, half precision, head dim 64
        _case("write_ragged_f16", "write", "1,733,1,1,2049,0,17,1", "500,0,33,4095,1000,12,70,9", kv_heads=12, dim=64,
              page=32, dtype="f16", store="e4m3"),
        # the 8-bit cache of four conversations turned into plain tensors (for an operator that takes those)
        _case("read_long_e4m3", "read", "1,1,1,1", "8191,4000,6143,8190", kv_heads=32, store="e4m3", page=64),
        # short, 16 bits, odd lengths
        _case("read_short", "read", "1,1,1", "200,517,33", kv_heads=8, dim=64, dtype="f16"),
        # a generation step of one conversation: latency
        _case("decode_one", "attn", "1", "999", lse=True),
        # one long conversation, 32 key / value heads, 8 bits
        _case("decode_long_e4m3", "attn", "1", "65535", kv_heads=32, store="e4m3", page=64),
        # a generation step of 16 conversations of unequal length, 4 query heads to a key / value head
        _case("decode_batch", "attn", _texts([1] * 16),
              "32767,900,16000,31001,8191,24575,12000,32000,4100,20480,28000,15,30011,6200,18000,26001", page=64),
        # checking five drafted tokens per sequence under a sliding window
        _case("verify_window_f16", "attn", _texts([5] * 8), "4000,1019,77,2500,8000,3,1300,6001", dim=64, dtype="f16",
              window=1024, page=32, lse=True),
        # a chunk of 2048 tokens of a long prompt
        _case("chunk_long", "attn", "2048", "8192", page=64),
        # a short chunk at the end of a long 16-bit cache: few rows, many keys
        _case("chunk_short", "attn", "61", "32707", page=64, lse=True),
        # continuous batching over the 8-bit cache: chunks and single tokens in one call
        _case("mixed_e4m3", "attn", "1024,1,311,1,1,130,1,1", "2048,4000,0,1777,350,3000,4090,12", kv_heads=32,
              store="e4m3"),
    ]


_MOST = {"bytes": 1.0e9, "flops": 3.0e11, "scores": 7.0e8, "rows": 6.0e8}


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(["write", "read", "attn", "attn", "attn"])
        kv_heads = rng.choice([1, 2, 5, 8, 8, 12, 32])
        group = rng.choice([1, 2, 4, 7, 8]) if kv_heads <= 8 else 1
        seqs = spread(1, 64)
        longest = spread(16, 65536)
        past = [rng.randint(longest // 8, longest) if rng.random() < 0.8 else rng.randint(0, longest // 8)
                for _ in range(seqs)]
        kind = rng.choice(["single", "few", "chunk", "mixed"])
        most = {"single": 1, "few": 8, "chunk": 8192 if op == "write" else 4096, "mixed": 2048}[kind]
        top = spread(max(1, most // 64), most)
        new = [rng.randint(1, top) if (kind in ("few", "chunk") or rng.random() < 0.25) else 1 for _ in range(seqs)]
        store = rng.choice(["same", "e4m3"]) if op != "write" or rng.random() < 0.3 else "e4m3"
        causal = op != "attn" or rng.random() < 0.9
        window = spread(1, 4096) if op == "attn" and causal and rng.random() < 0.3 else -1
        case = _case("", op, _texts(new), _texts(past), heads=kv_heads * group, kv_heads=kv_heads,
                     dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128, 256]),
                     dtype=rng.choice(["bf16", "bf16", "f16"]), store=store, window=window, causal=causal,
                     lse=op == "attn" and rng.random() < 0.4)
        del case["name"]
        w = work(case)
        total = max(p + n for p, n in zip(past, new))
        rows = seqs * total * kv_heads * case["dim"]
        scores = seqs * total * max(new) * case["heads"] if op == "attn" else 0
        if w["bytes"] <= _MOST["bytes"] and w["flops"] <= _MOST["flops"] and scores <= _MOST["scores"] and rows <= _MOST["rows"]:
            return case


def _lengths(case):
    new = [int(x) for x in case["new"].split(",")]
    past = [int(x) for x in case["past"].split(",")]
    return new, past


def _visible(case, n, p):
    """(row, key) pairs a sequence of n new rows behind p cached ones scores, and the keys it touches."""
    if not case["causal"]:
        return n * (n + p), n + p
    w = case["window"]
    if w < 0:
        return n * p + n * (n + 1) // 2, n + p
    pairs = sum(min(p + t, w) + 1 for t in range(n))
    return pairs, min(n + p, w + n)


def work(case):
    new, past = _lengths(case)
    dim, kvh = case["dim"], case["kv_heads"]
    row16 = 2 * dim
    row = dim + 1 if case["store"] == "e4m3" else row16
    if case["op"] == "write":
        return {"bytes": sum(new) * kvh * 2 * (row16 + row), "flops": 0}
    if case["op"] == "read":
        n_out = max(n + p for n, p in zip(new, past))
        return {"bytes": sum(n + p for n, p in zip(new, past)) * kvh * 2 * row + len(new) * n_out * kvh * 2 * row16,
                "flops": 0}
    pairs = keys = 0
    for n, p in zip(new, past):
        a, b = _visible(case, n, p)
        pairs, keys = pairs + a, keys + b
    n_bytes = keys * kvh * 2 * row + sum(new) * case["heads"] * (2 * row16 + (4 if case["lse"] else 0))
    return {"bytes": n_bytes, "flops": 4 * case["heads"] * dim * pairs}


# ---------------------------------------------------------------------------------------------------------------------
def _exponents(x):
    """Byte of the smallest power of two that brings each row of x (fp32, last dimension) into e4m3's +-448."""
    top = x.abs().amax(-1)
    frac, exp = torch.frexp(top)  # top = frac * 2^exp, frac in [0.5, 1)
    e = exp - 9 + (frac > 0.875)
    return torch.where(top > 0, e.clamp(-126, 120), torch.full_like(e, -126)) + 127


def _power(e):
    """2^e, exactly, for whole numbers -126 <= e <= 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    byte = _exponents(x)
    return (x * _power(127 - byte).unsqueeze(-1)).to(E4M3), byte.to(torch.uint8)


def _top(dtype):
    return 1.875 * 2.0 ** (15 if dtype == torch.float16 else 127)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    dtype = TYPES[case["dtype"]]
    new, past = _lengths(case)
    heads, kvh, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    S, T = len(new), sum(new)
    lens = [n + p for n, p in zip(new, past)]
    need = [-(-n // page) for n in lens]
    width = max(need)
    n_pages = sum(need) + 3  # a few pages that nobody owns

    # the block table: every sequence's pages lie anywhere in the pool; entries behind its last page are -1
    order = torch.randperm(n_pages, generator=g, device=dev)[: sum(need)].to(torch.int32)
    held = torch.tensor(need, device=dev)
    cells = torch.arange(width, device=dev)[None] < held[:, None]
    table = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    table[cells] = order

    # a few channels of the keys are several times the others, as in trained models
    loud = torch.ones(dim, device=dev)
    loud[torch.randperm(dim, generator=g, device=dev)[: max(1, dim // 32)]] = 3.0

    def pool(scale):
        quantised = case["store"] == "e4m3"
        pages = torch.empty((n_pages, kvh, page, dim), dtype=E4M3 if quantised else dtype, device=dev)
        exps = torch.empty((n_pages, kvh, page), dtype=torch.uint8, device=dev) if quantised else None
        step = max(1, (1 << 25) // (kvh * page * dim))
        for a in range(0, n_pages, step):
            b = min(n_pages, a + step)
            x = torch.randn((b - a, kvh, page, dim), generator=g, device=dev) * scale
            if quantised:
                q, e = _quantise(x)
                pages.view(torch.uint8)[a:b] = q.view(torch.uint8)
                exps[a:b] = e
            else:
                pages[a:b] = x.to(dtype)
        return pages, exps

    k_pages, k_exp = pool(loud)
    v_pages, v_exp = pool(1.0)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {"case": dict(case), "k_pages": k_pages, "v_pages": v_pages, "k_exp": k_exp, "v_exp": v_exp, "table": table,
             "cu": torch.tensor(starts, dtype=torch.int32, device=dev),
             "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "max_q": max(new), "max_len": max(lens),
             "dtype": dtype}
    if case["op"] != "read":  # the projection's output, one buffer of query, key and value columns
        qkv = torch.randn((T, (heads + 2 * kvh) * dim), generator=g, device=dev)
        qkv[:, heads * dim : (heads + kvh) * dim] *= loud.repeat(kvh)
        qkv = qkv.to(dtype)
        state["q"] = qkv[:, : heads * dim].view(T, heads, dim)
        state["k"] = qkv[:, heads * dim : (heads + kvh) * dim].view(T, kvh, dim)
        state["v"] = qkv[:, (heads + kvh) * dim :].view(T, kvh, dim)
    return state


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms.
def _rows_of(state):
    """Sequence and place among the sequence's new rows of each packed row."""
    cu = state["cu"].long()
    t = torch.arange(state["q"].shape[0], device=cu.device)
    s = torch.searchsorted(cu, t, right=True) - 1
    return s, t - cu[s]


def _plain_write(state):
    case, table = state["case"], state["table"]
    page = case["page"]
    s, t = _rows_of(state)
    cu, lens = state["cu"].long(), state["lens"].long()
    pos = lens[s] - (cu[s + 1] - cu[s]) + t
    at, off = table[s, pos // page].long(), pos % page
    outs = []
    for x, pages, exps in ((state["k"], state["k_pages"], state["k_exp"]), (state["v"], state["v_pages"], state["v_exp"])):
        if exps is None:
            pages[at, :, off] = x
            outs.append(pages)
        else:
            top = _top(state["dtype"])
            q, e = _quantise(x.float().clamp(-top, top))
            pages.view(torch.uint8)[at, :, off] = q.view(torch.uint8)
            exps[at, :, off] = e
            outs += [pages, exps]
    return outs


def _values(pages, exps, table, n):
    """[S, kv_heads, n, dim] in 32 bits: the first n rows of every sequence."""
    at = table.clamp(min=0).long()
    if exps is None:
        x = pages[at].float()
    else:
        x = pages.view(torch.uint8)[at].view(E4M3).float() * _power(exps[at].int() - 127).unsqueeze(-1)
    S, width, kvh, page, dim = x.shape
    return x.transpose(1, 2).reshape(S, kvh, width * page, dim)[:, :, :n]


def _plain_read(state):
    n = state["max_len"]
    live = (torch.arange(n, device=state["lens"].device)[None] < state["lens"][:, None])[:, None, :, None]
    k = _values(state["k_pages"], state["k_exp"], state["table"], n)
    v = _values(state["v_pages"], state["v_exp"], state["table"], n)
    zero = torch.zeros((), device=k.device)
    return [torch.where(live, k, zero).to(state["dtype"]), torch.where(live, v, zero).to(state["dtype"])]


def _plain_attn(state):
    case = state["case"]
    q, lens, cu = state["q"], state["lens"].long(), state["cu"].long()
    T, heads, dim = q.shape
    kvh = case["kv_heads"]
    S, mq, n = lens.numel(), state["max_q"], state["max_len"]
    s, t = _rows_of(state)
    k = _values(state["k_pages"], state["k_exp"], state["table"], n)
    v = _values(state["v_pages"], state["v_exp"], state["table"], n)
    rows = torch.zeros((S, mq, heads, dim), device=q.device)
    rows[s, t] = q.float()
    rows = rows.view(S, mq, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(S, kvh, -1, dim)
    scores = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(dim))
    scores = scores.view(S, heads, mq, n)
    j = torch.arange(n, device=q.device)
    seen = (j[None, :] < lens[:, None])[:, None, :]
    if case["causal"]:
        i = (lens - (cu[1:] - cu[:-1]))[:, None] + torch.arange(mq, device=q.device)[None]
        seen = seen & (j[None, None, :] <= i[:, :, None])
        if case["window"] >= 0:
            seen = seen & (i[:, :, None] - j[None, None, :] <= case["window"])
    scores.masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(S, kvh, -1, n), v).view(S, heads, mq, dim) / total
    out = out.permute(0, 2, 1, 3)[s, t].to(state["dtype"])
    if not case["lse"]:
        return [out]
    lse = ((top + total.log()) * LOG2E).squeeze(-1).permute(0, 2, 1)[s, t]
    return [out, lse]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn}[op](state)
    from vqtree_amd.ops import paged_cache

    case = state["case"]
    pools = (state["k_pages"], state["v_pages"])
    exps = {"k_exp": state["k_exp"], "v_exp": state["v_exp"]}
    if op == "write":
        paged_cache.paged_write(state["k"], state["v"], *pools, state["table"], state["cu"], state["lens"], **exps)
        return [x for x in (state["k_pages"], state["k_exp"], state["v_pages"], state["v_exp"]) if x is not None]
    if op == "read":
        return list(paged_cache.paged_read(*pools, state["table"], state["lens"], state["max_len"], dtype=state["dtype"],
                                           **exps))
    got = paged_cache.attn_paged(state["q"], *pools, state["table"], state["cu"], state["lens"], **exps,
                                 causal=case["causal"], window=case["window"] if case["window"] >= 0 else None,
                                 return_lse=case["lse"], max_q_len=state["max_q"])
    return list(got) if case["lse"] else [got]


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits.
def _two_to(e):
    """2^e in 64 bits, exactly (a power function may be off by a last place, which moves ties)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_stored(x):
    """e4m3 elements of rows x (64 bits): scaled by the row's power of two, rounded to the nearest of 4 significant bits."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0**-140)))
    e = torch.where(top < _two_to(e), e - 1, e)
    e = torch.where(top >= _two_to(e + 1), e + 1, e)
    e = torch.where(top > 1.75 * _two_to(e), e - 7, e - 8).clamp(-126, 120)
    y = x * _two_to(-e)
    size = torch.floor(torch.log2(y.abs().clamp(min=2.0**-6)))
    size = torch.where(y.abs() >= _two_to(size + 1), size + 1, size)
    size = torch.where((y.abs() < _two_to(size)) & (size > -6), size - 1, size)
    return torch.round(y * _two_to(3 - size)) * _two_to(size - 3)


def exact(case, seed):
    state = prepare(case, seed)
    new, past = _lengths(case)
    page, dim, kvh, heads = case["page"], case["dim"], case["kv_heads"], case["heads"]
    table = state["table"].tolist()
    pools = [(state["k_pages"], state["k_exp"]), (state["v_pages"], state["v_exp"])]
    if case["op"] == "write":
        outs = []
        for (pages, exps), x in zip(pools, (state["k"], state["v"])):
            want = pages.double()
            r = 0
            for s, (n, p) in enumerate(zip(new, past)):
                if n == 0:
                    continue
                rows = x[r : r + n].double()
                if exps is not None:
                    rows = _exact_stored(rows)
                where = torch.tensor([[table[s][i // page], i % page] for i in range(p, p + n)], device=rows.device)
                want[where[:, 0], :, where[:, 1]] = rows
                r += n
            outs += [want] if exps is None else [want, None]
        return outs

    def rows_of(s, pages, exps, n, h=slice(None)):
        ids = torch.tensor(table[s][: -(-n // page)], device=pages.device)
        x = pages[ids][:, h].double() if exps is None else pages.view(torch.uint8)[ids][:, h].view(E4M3).double()
        if exps is not None:
            x = x * _two_to(exps[ids][:, h].long() - 127).unsqueeze(-1)
        return x.transpose(0, 1).reshape(x.shape[1], -1, dim)[:, :n]

    if case["op"] == "read":
        outs = [torch.zeros((len(new), kvh, state["max_len"], dim), dtype=torch.float64, device="cuda") for _ in pools]
        for want, (pages, exps) in zip(outs, pools):
            for s, (n, p) in enumerate(zip(new, past)):
                want[s, :, : n + p] = rows_of(s, pages, exps, n + p)
        return outs

    group = heads // kvh
    out = torch.zeros((sum(new), heads, dim), dtype=torch.float64, device="cuda")
    lse = torch.zeros((sum(new), heads), dtype=torch.float64, device="cuda")
    r = 0
    for s, (n, p) in enumerate(zip(new, past)):
        j = torch.arange(n + p, device="cuda")
        i = torch.arange(p, p + n, device="cuda")[:, None]
        hidden = torch.zeros((n, n + p), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden = j > i
            if case["window"] >= 0:
                hidden = hidden | (j < i - case["window"])
        for h in range(kvh):
            k = rows_of(s, *pools[0], n + p, slice(h, h + 1))[0]
            v = rows_of(s, *pools[1], n + p, slice(h, h + 1))[0]
            for c in range(h * group, (h + 1) * group):
                z = state["q"][r : r + n, c].double() @ k.t() / math.sqrt(dim)
                z = z.masked_fill(hidden, -math.inf)
                l = torch.logsumexp(z, -1)
                out[r : r + n, c] = torch.exp(z - l[:, None]) @ v
                lse[r : r + n, c] = l / math.log(2.0)
        r += n
    return [out, lse] if case["lse"] else [out]


if __name__ == "__main__":
    rng = random.Random(0)
    for c in listed() + [draw(rng) for _ in range(20)]:
        w = work(c)
        print("%-20s %-6s %10.3f MB %10.3f GFLOP" % (c.get("name", "(drawn)"), c["op"], w["bytes"] / 1e6, w["flops"] / 1e9))
