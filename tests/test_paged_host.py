"""Paged cache, CPU side: the 64-bit oracle against independent statements, and what the entry points refuse."""
import math
import os
import subprocess
import sys

import pytest
import torch

from oracle import paged as O
from vqtree_amd import _lib
from vqtree_amd.ops import paged_cache as P

ERRORS = (AssertionError, _lib.VqaError)


def test_oracle_quantiser_is_the_cast_of_the_scaled_row():
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(5, 3, 64, generator=g) * torch.tensor([1e-3, 1.0, 300.0]).view(1, 3, 1)).to(torch.bfloat16)
    x[0, 0] = 0
    x[1, 1, :4] = torch.tensor([448.0, 449.0, -480.0, 2.0**-12])
    values, byte = O.quantise_rows(x)
    scaled = torch.ldexp(x.float(), 127 - byte.int().unsqueeze(-1))
    assert float(scaled.abs().max()) <= 448.0
    back = torch.ldexp(scaled.to(torch.float8_e4m3fn).float(), byte.int().unsqueeze(-1) - 127)
    assert torch.equal(back.double(), values)
    assert int(byte[0, 0]) == 1


@pytest.mark.parametrize("causal", [True, False])
def test_oracle_attention_equals_dense_softmax(causal):
    g = torch.Generator().manual_seed(1)
    H, G, D, page, n_keys, n = 2, 3, 64, 16, 45, 7
    pages = torch.randn(2, 6, H, page, D, generator=g, dtype=torch.float64)
    table = torch.tensor([[4, 0, 2]], dtype=torch.int32)
    q = torch.randn(n, H * G, D, generator=g, dtype=torch.float64)
    out, lse, _, _ = O.paged_attention(q, pages[0], pages[1], table, torch.tensor([0, n]), torch.tensor([n_keys]), causal=causal)
    k, v = (p[[4, 0, 2]].transpose(0, 1).reshape(H, -1, D)[:, :n_keys].repeat_interleave(G, 0) for p in pages)
    mask = torch.ones(n, n_keys, dtype=torch.bool)
    if causal:
        mask = mask.tril(n_keys - n)
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1)[None], k[None], v[None], attn_mask=mask)[0]
    assert torch.allclose(out.transpose(0, 1), want, atol=1e-12)
    assert torch.isfinite(lse).all()


def _call(**change):
    H, D, page, n_pages, S, T = 2, 64, 16, 3, 2, 4
    a = dict(q=torch.zeros(T, 4, D, dtype=torch.bfloat16), k_pages=torch.zeros(n_pages, H, page, D, dtype=torch.bfloat16),
             v_pages=torch.zeros(n_pages, H, page, D, dtype=torch.bfloat16),
             block_table=torch.zeros(S, 2, dtype=torch.int32), cu_q=torch.zeros(S + 1, dtype=torch.int32),
             kv_lens=torch.zeros(S, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(4, 3, 64, dtype=torch.bfloat16)),                 # 3 query heads for 2 key heads
    dict(q=torch.zeros(4, 4, 128, dtype=torch.bfloat16)),                # another head dim
    dict(q=torch.zeros(4, 4, 64, dtype=torch.float16)),                  # another type than the pages
    dict(q=torch.zeros(4, 4, 64)),                                       # fp32
    dict(q=torch.zeros(1, 4, 4, 64, dtype=torch.bfloat16)),
    dict(block_table=torch.zeros(2, 2, dtype=torch.int64)),
    dict(block_table=torch.zeros(2, 0, dtype=torch.int32)),
    dict(kv_lens=torch.zeros(3, dtype=torch.int32)),
    dict(cu_q=torch.zeros(2, dtype=torch.int32)),
    dict(cu_q=torch.zeros(3, dtype=torch.int64)),
    dict(window=-1),
    dict(window=5, causal=False),
    dict(softmax_scale=-1.0),
    dict(k_exp=torch.zeros(3, 2, 16, dtype=torch.uint8), v_exp=torch.zeros(3, 2, 16, dtype=torch.uint8)),
    dict(out=torch.zeros(4, 4, 64)),
    dict(k_pages=torch.zeros(3, 2, 24, 64, dtype=torch.bfloat16), v_pages=torch.zeros(3, 2, 24, 64, dtype=torch.bfloat16)),
    dict(k_pages=torch.zeros(3, 2, 16, 64, dtype=torch.float8_e4m3fn), v_pages=torch.zeros(3, 2, 16, 64, dtype=torch.float8_e4m3fn)),
    dict(k_pages=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)),
])
def test_attention_refuses(change):
    with pytest.raises(AssertionError):
        P.attn_paged(**_call(**change))


def test_write_and_read_refuse():
    a = _call()
    k = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    tail = (a["k_pages"], a["v_pages"], a["block_table"], a["cu_q"], a["kv_lens"])
    for bad in (k[:, :1], k.half(), k[..., :32], k[0]):
        with pytest.raises(AssertionError):
            P.paged_write(bad, bad, *tail)
    with pytest.raises(AssertionError):
        P.paged_write(k, k[:3], *tail)
    with pytest.raises(AssertionError):
        P.paged_read(a["k_pages"], a["v_pages"], a["block_table"], a["kv_lens"], -1)
    with pytest.raises(AssertionError):  # 8-bit pages say nothing of the type to read them as
        e8 = torch.zeros(3, 2, 16, 64, dtype=torch.float8_e4m3fn)
        e = torch.zeros(3, 2, 16, dtype=torch.uint8)
        P.paged_read(e8, e8, a["block_table"], a["kv_lens"], 4, k_exp=e, v_exp=e)
    # everything in order but for the device: there is no CPU path
    with pytest.raises(_lib.VqaError):
        P.attn_paged(**a)
    with pytest.raises(_lib.VqaError):
        P.paged_write(k, k, *tail)
    with pytest.raises(_lib.VqaError):
        P.paged_read(a["k_pages"], a["v_pages"], a["block_table"], a["kv_lens"], 4)


def test_c_entries_refuse_before_any_launch(lib):
    st = _lib.strides_array(*([128] * 17))
    ok = dict(T=4, S=2, Hq=4, Hkv=2, D=64, page=16, n_pages=3, width=2, e4m3=0, causal=1, window=-1, scale=1.0, q=16, exp=16)

    def attn(**kw):
        a = dict(ok, **kw)
        need = lib.vqa_paged_attn_workspace_bytes(a["T"], a["S"], a["Hq"], a["Hkv"], a["D"], a["page"], a["width"], a["e4m3"], a["causal"],
                                                  a["window"], a["T"])
        ws = kw.get("ws", need)
        return lib.vqa_paged_attn_bf16(a["q"], 16, 16, a["exp"], a["exp"], 16, 16, 16, 16, None, 256, ws, a["T"], a["S"],
                                       a["Hq"], a["Hkv"], a["D"], a["page"], a["n_pages"], a["width"], a["e4m3"], st,
                                       a["causal"], a["window"], a["T"], a["scale"], None)

    assert attn(q=None) == -1 and attn(e4m3=1, exp=None) == -1
    assert attn(Hq=3) == -2 and attn(Hkv=0) == -2 and attn(T=-1) == -2 and attn(width=0) == -2 and attn(n_pages=0) == -2
    assert attn(width=1 << 27) == -2  # more keys than 2^30
    assert attn(D=96) == -3
    assert attn(q=24) == -5
    assert attn(page=8) == -7 and attn(page=48) == -7 and attn(page=8192) == -7
    assert attn(window=4, causal=0) == -7 and attn(scale=0.0) == -7 and attn(scale=math.nan) == -7
    assert attn(T=0) == 0 and attn(S=0) == 0  # nothing to do: nothing is launched

    def write(**kw):
        a = dict(ok, **kw)
        return lib.vqa_paged_write_f16(a["q"], 16, 16, 16, a["exp"], a["exp"], 16, 16, 16, a["T"], a["S"], a["Hkv"], a["D"],
                                       a["page"], a["n_pages"], a["width"], a["e4m3"], st, None)

    assert write(q=None) == -1 and write(e4m3=1, exp=None) == -1 and write(D=32) == -3 and write(page=17) == -7
    assert write(q=8) == -5 and write(Hkv=0) == -2 and write(S=0) == 0

    def read(**kw):
        a = dict(ok, n=5, **kw) if "n" not in kw else dict(ok, **kw)
        return lib.vqa_paged_read_f16(16, 16, a["exp"], a["exp"], 16, 16, a["q"], 16, a["S"], a["Hkv"], a["n"], a["D"],
                                      a["page"], a["n_pages"], a["width"], a["e4m3"], st, None)

    assert read(q=None) == -1 and read(S=1 << 17) == -2 and read(n=-1) == -2 and read(q=8) == -5 and read(n=0) == 0
    bad = _lib.strides_array(*([4] * 17))
    assert lib.vqa_paged_read_f16(16, 16, None, None, 16, 16, 16, 16, 2, 2, 5, 64, 16, 3, 2, 0, bad, None) == -5


def test_numbers_given_as_tensors_are_read_at_every_call(lib, monkeypatch):
    """What is kept of a call follows from values: a window, a hint or a number of rows held in a tensor counts as it is now."""
    calls = []
    monkeypatch.setattr(P, "_check_devices", lambda *a: None)
    monkeypatch.setattr(P, "_launch", lambda fn, dev, *a: calls.append(a))
    a = _call()
    n, window, longest, scale = torch.tensor(30), torch.tensor(20), torch.tensor(4), torch.tensor(0.5)
    for _ in range(2):
        k, v = P.paged_read(a["k_pages"], a["v_pages"], a["block_table"], a["kv_lens"], n)
        S, H, rows, D = calls[-1][8:12]
        strides = list(calls[-1][-1])
        assert (S, H, rows, D) == tuple(k.shape) == tuple(v.shape) == (2, 2, int(n), 64)
        assert strides[11:14] == list(k.stride()[:3]) and strides[14:] == list(v.stride()[:3])
        P.attn_paged(**a, window=window, max_q_len=longest, softmax_scale=scale)
        causal, w, max_q, s = calls[-1][-4:]
        assert (causal, w, max_q, s) == (1, int(window), int(longest), float(scale))
        n.fill_(4), window.fill_(3), longest.fill_(1), scale.fill_(0.25)
    with pytest.raises(TypeError):
        P.paged_read(a["k_pages"], a["v_pages"], a["block_table"], a["kv_lens"], 4.0)


# A HIP runtime of two devices that launches nothing: every pointer lies on `owner`.
RUNTIME = """
#include <string.h>
typedef struct { int type, device; void *device_pointer, *host_pointer; int managed; unsigned flags; } attributes;
typedef struct { unsigned x, y, z; } dim3_t;
int current = 0, owner = 0, launches = 0;
int hipGetDevice(int* d) { *d = current; return 0; }
int hipPointerGetAttributes(attributes* a, const void* p) {
    memset(a, 0, sizeof *a);
    a->type = 2, a->device = owner, a->device_pointer = (void*)p;
    return 0;
}
int hipFuncSetAttribute(const void* f, int a, int v) { return 0; }
int hipGetLastError(void) { return 0; }
int hipLaunchKernel(const void* f, dim3_t g, dim3_t b, void** args, size_t lds, void* stream) { ++launches; return 0; }
int __hipPushCallConfiguration(dim3_t g, dim3_t b, size_t lds, void* stream) { return 0; }
int __hipPopCallConfiguration(dim3_t* g, dim3_t* b, size_t* lds, void** stream) {
    g->x = g->y = g->z = b->x = b->y = b->z = 1, *lds = 0, *stream = 0;
    return 0;
}
"""

TWO_DEVICES = """
import ctypes, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # (found before the runtime the library brings with it)
sys.path.insert(0, sys.argv[2])
from vqtree_amd import _lib
lib = _lib.load()
number = lambda name: ctypes.c_int.in_dll(stub, name)
st = _lib.strides_array(*([128] * 17))

def attn(T, S, Hkv, D, width):
    need = lib.vqa_paged_attn_workspace_bytes(T, S, Hkv, Hkv, D, 16, width, 0, 1, -1, T)
    return lib.vqa_paged_attn_bf16(16, 16, 16, None, None, 16, 16, 16, 16, None, 256, need, T, S, Hkv, Hkv, D, 16, 3, width,
                                   0, st, 1, -1, T, 1.0, None)

calls = {
    "single token": lambda: attn(1, 1, 2, 128, 8),
    "single tokens, narrow workgroups": lambda: attn(300, 300, 2, 128, 8),
    "chunk": lambda: attn(512, 1, 2, 64, 16384),
    "chunk, head dim 128": lambda: attn(512, 1, 2, 128, 16384),
    "write": lambda: lib.vqa_paged_write_bf16(16, 16, 16, 16, None, None, 16, 16, 16, 4, 2, 2, 64, 16, 3, 2, 0, st, None),
    "read": lambda: lib.vqa_paged_read_bf16(16, 16, None, None, 16, 16, 16, 16, 2, 2, 5, 64, 16, 3, 2, 0, st, None),
}
for turn in range(2):  # (the second time everything is set up on both devices)
    for name, call in calls.items():
        for device in (0, 1):
            for owner in (0, 1):
                number("current").value, number("owner").value, number("launches").value = device, owner, 0
                rc, n = call(), number("launches").value
                good = (rc == 0 and n > 0) if device == owner else (rc == -7 and n == 0)
                if not good:
                    print(name, "turn", turn, "device", device, "owner", owner, "status", rc, "launches", n)
print("done")
"""


def test_operands_of_another_device_are_refused_at_every_call(tmp_path, lib):
    source, stub = tmp_path / "runtime.c", tmp_path / "runtime.so"
    source.write_text(RUNTIME)
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-include", "stddef.h", str(source), "-o", str(stub)], check=True)
    root = os.path.dirname(os.path.dirname(os.path.abspath(P.__file__)))
    got = subprocess.run([sys.executable, "-c", TWO_DEVICES, str(stub), os.path.dirname(root)], capture_output=True, text=True,
                         timeout=120)
    assert got.returncode == 0, got.stderr
    assert got.stdout == "done\n", got.stdout
