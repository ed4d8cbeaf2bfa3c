"""The 8-bit cache's host side (no GPU): rounding to codes, and what the calls refuse.

A value x of a row whose largest magnitude is a is kept as code * (a / top).
With exact arithmetic it would be within half a code step: a / 254 for int8;
for e4m3 half the spacing of four significant bits, 2^-4 |x| at most, or half
of its smallest step 2^-9.  The fp32 products before and after (a / top, top / a,
x times that, code times scale) are each off by a relative 2^-24; together they
move a value, or the tie it is rounded at, by less than 2^-21 of a.
"""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from vllm_mps_b200 import kernels as K

FORMATS = [torch.int8, torch.float8_e4m3fn]


def _half_step(x, fmt):
    a = x.abs().amax(-1, keepdim=True)
    if fmt == torch.int8:
        return a / 254 + a * 2.0 ** -21
    return torch.maximum(x.abs() * 2.0 ** -4, a / 448 * 2.0 ** -10) + a * 2.0 ** -21


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e4, 1.0, 1e-4, 1e-25])
def test_values_are_within_half_a_step(size, fmt):
    g = torch.Generator().manual_seed(1)
    x = torch.randn((64, 128), generator=g) * size
    x[3] *= torch.rand(128, generator=g) ** 8  # a few large channels
    x[5] = 0
    codes, scales = K.quantize_cache8(x, fmt)
    assert codes.dtype == fmt and scales.shape == (64,) and scales[5] == 0
    got = codes.double() * scales.double().unsqueeze(1)
    assert ((got - x.double()).abs() <= _half_step(x.double(), fmt)).all()
    top = codes.float().abs().amax(1)
    assert (top[torch.arange(64) != 5] == K._CACHE_TOP[fmt]).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_are_no_numbers_or_tiny(fmt):
    x = torch.ones((6, 64))
    x[0, 3], x[1, 63], x[2, 0] = float("nan"), float("inf"), -float("inf")
    x[3] = 2.0 ** -101
    x[4] = 2.0 ** -100
    codes, scales = K.quantize_cache8(x, fmt)
    assert torch.isnan(scales[:3]).all() and (codes[:4].float() == 0).all()
    assert scales[3] == 0
    for row in (4, 5):
        got = codes[row].float() * scales[row]
        assert ((got - x[row]).abs() <= x[row] * 2.0 ** -21).all()


def test_cache_layout_and_dequantize():
    c = K.KVCache8.zeros(3, 2, 64, torch.int8, device="cpu")
    assert c.codes.shape == (3, 2, 16, 2, 64) and c.scales.shape == (3, 2, 2, 16)
    c.codes[1, 1, 5, 0, 7] = -9
    c.scales[1, 0, 1, 5] = 0.5
    full = c.dequantize()
    assert full[1, 1, 5, 0, 7] == -4.5 and full.abs().sum() == 4.5


def test_caches_that_are_refused():
    codes = torch.zeros((3, 2, 16, 2, 64), dtype=torch.int8)
    scales = torch.zeros((3, 2, 2, 16))
    with pytest.raises(TypeError):
        K.KVCache8(codes.half(), scales)
    with pytest.raises(TypeError):
        K.KVCache8(codes.to(torch.float8_e5m2), scales)
    for bad in (codes[:, :1], codes[:, :, :8], codes[0], codes.transpose(3, 4)):
        with pytest.raises(ValueError):
            K.KVCache8(bad, scales)
    for bad in (scales.double(), scales[:2], scales.transpose(0, 1), scales.transpose(1, 2)):
        with pytest.raises(ValueError):
            K.KVCache8(codes, bad)
    with pytest.raises(TypeError):
        K.quantize_cache8(torch.zeros(4), torch.uint8)


def _store_args(rows=3, n_q=4, n_kv=2, D=64, dtype=torch.float16):
    return dict(q=torch.zeros((rows, n_q, D), dtype=dtype), k=torch.zeros((rows, n_kv, D), dtype=dtype),
                v=torch.zeros((rows, n_kv, D), dtype=dtype),
                positions=torch.zeros(rows, dtype=torch.int32),
                slot_mapping=torch.zeros(rows, dtype=torch.int32),
                inv_freq=torch.ones(D // 2), cache=K.KVCache8.zeros(2, n_kv, D, device="cpu"))


@pytest.mark.parametrize("change, error", [
    (dict(k=torch.zeros((3, 2, 64), dtype=torch.bfloat16)), TypeError),
    (dict(cache=torch.zeros((2, 2, 16, 2, 64), dtype=torch.bfloat16)), TypeError),
    (dict(cache=torch.zeros((2, 16, 2, 64), dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros((3, 3, 64), dtype=torch.float16)), ValueError),
    (dict(v=torch.zeros((4, 2, 64), dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros((2, 4, 64), dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros((3, 64, 4), dtype=torch.float16).transpose(1, 2)), ValueError),
    (dict(q_out=torch.zeros((3, 5, 64), dtype=torch.float16)), ValueError),
    (dict(q=None, q_out=torch.zeros((3, 4, 64), dtype=torch.float16)), ValueError),
    (dict(positions=None), ValueError),
    (dict(positions=torch.zeros(3)), TypeError),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(slot_mapping=torch.zeros(6, dtype=torch.int32)[::2]), ValueError),
    (dict(inv_freq=torch.ones(64)), ValueError),
    (dict(q_weight=torch.ones(64)), ValueError),
    (dict(k_weight=torch.ones(32, dtype=torch.float16)), ValueError),
    (dict(), RuntimeError),  # host tensors: there is no CPU path
])
def test_store_refusals(change, error):
    with pytest.raises(error):
        K.norm_rope_and_cache(**{**_store_args(), **change})


_Q = torch.zeros((3, 4, 64), dtype=torch.float16)


@pytest.mark.parametrize("change, error", [
    (dict(q=torch.zeros((3, 4, 32), dtype=torch.float16)), ValueError),
    (dict(block_tables=torch.zeros((2, 5), dtype=torch.int32)), ValueError),
    (dict(block_tables=torch.zeros((3, 5), dtype=torch.int64)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(out=torch.zeros((3, 4, 64), dtype=torch.bfloat16)), ValueError),
    (dict(out=_Q, q=_Q), ValueError),
    (dict(), RuntimeError),
])
def test_decode_refusals(change, error):
    args = dict(q=torch.zeros((3, 4, 64), dtype=torch.float16), cache=K.KVCache8.zeros(2, 2, 64, device="cpu"),
                block_tables=torch.zeros((3, 5), dtype=torch.int32),
                seq_lens=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(error):
        K.paged_decode_attention_cache8(**{**args, **change})


@pytest.mark.parametrize("change, error", [
    (dict(pool=torch.zeros((4, 2, 16, 2, 128), dtype=torch.float16)), ValueError),
    (dict(dst_tables=torch.zeros((3, 4), dtype=torch.int32)), ValueError),
    (dict(dst_tables=torch.zeros((3, 5), dtype=torch.int64)), TypeError),
    (dict(seq_lens=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(), RuntimeError),
])
def test_read_refusals(change, error):
    args = dict(cache=K.KVCache8.zeros(2, 2, 64, device="cpu"),
                block_tables=torch.zeros((3, 5), dtype=torch.int32),
                seq_lens=torch.zeros(3, dtype=torch.int32),
                pool=torch.zeros((4, 2, 16, 2, 64), dtype=torch.float16),
                dst_tables=torch.zeros((3, 5), dtype=torch.int32))
    with pytest.raises(error):
        K.read_cache8(**{**args, **change})


# The C entries check everything on the host before they touch the device: the
# addresses below are never read.
A = 1 << 20


def _lib():
    if not os.path.exists(K.LIB_PATH):
        pytest.skip("library not built")
    return K.load_library()


def _c_store(**change):
    a = dict(q_out=A, qos=256, q=A, qs=256, k=A, ks=128, v=A, vs=128, qw=A, kw=A, eps=1e-6, pos=A,
             slot=A, inv=A, cache=A, scales=A, rows=3, n_q=4, n_kv=2, d=64, bs=16, nb=2,
             fmt=K.VMPS_CACHE_INT8, dtype=0, stream=None)
    a.update(change)
    return _lib().vmps_norm_rope_and_cache(*a.values())


@pytest.mark.parametrize("change, rc", [
    (dict(rows=0), 0), (dict(rows=-1), -1), (dict(n_kv=0), -1), (dict(n_q=-1), -1), (dict(nb=0), -1),
    (dict(dtype=2), -1), (dict(fmt=3), -1), (dict(fmt=-1), -1), (dict(d=96), -2), (dict(d=256), -2),
    (dict(bs=32), -2), (dict(q=None), -1), (dict(q_out=None), -1), (dict(k=None), -1),
    (dict(v=None), -1), (dict(cache=None), -1), (dict(slot=None), -1), (dict(pos=None), -1),
    (dict(scales=None), -1), (dict(q=A + 8), -3), (dict(k=A + 2), -3), (dict(cache=A + 4), -3),
    (dict(qw=A + 2), -3), (dict(qs=257), -3), (dict(vs=132), -3), (dict(qs=248), -1),
    (dict(vs=120), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(scales=A + 2), -3),
])
def test_c_store_refusals(change, rc):
    assert _c_store(**change) == rc
    assert bool(_lib().vmps_last_error()) == (rc != 0)


@pytest.mark.parametrize("change, rc", [
    (dict(B=0), 0), (dict(B=-1), -1), (dict(B=4097), -2), (dict(nb=0), -1), (dict(mb=0), -1),
    (dict(dtype=2), -1), (dict(fmt=0), -1), (dict(d=96), -2), (dict(bs=8), -2), (dict(n_q=34), -2),
    (dict(n_q=3), -2), (dict(n_q=130, n_kv=65), -2), (dict(q=None), -1), (dict(out=None), -1),
    (dict(codes=None), -1), (dict(scales=None), -1), (dict(bt=None), -1), (dict(lens=None), -1),
    (dict(q=A + 2), -3), (dict(out=A + 2), -3), (dict(codes=A + 8), -3), (dict(scales=A + 4), -3),
    (dict(qs=260), -3), (dict(qs=248), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(B=4096, mb=1 << 17), -2), (dict(mb=1 << 27), -2),
    (dict(nb=1 << 30), -2),
])
def test_c_decode_refusals(change, rc):
    a = dict(out=A, q=A, qs=256, codes=A, scales=A, bt=A, mb=4, lens=A, B=3, n_q=4, n_kv=2, d=64,
             bs=16, nb=2, scale=0.125, ws=A, wsb=1 << 40, fmt=K.VMPS_CACHE_INT8, dtype=0, stream=None)
    a.update(change)
    assert _lib().vmps_paged_decode_attention_cache8(*a.values()) == rc


@pytest.mark.parametrize("change, rc", [
    (dict(B=0), 0), (dict(B=-1), -1), (dict(B=4097), -2), (dict(nb=0), -1), (dict(pb=0), -1),
    (dict(mb=0), -1), (dict(n_kv=65), -1), (dict(dtype=2), -1), (dict(fmt=0), -1), (dict(d=96), -2),
    (dict(bs=8), -2), (dict(pool=None), -1), (dict(dst=None), -1), (dict(codes=None), -1),
    (dict(scales=None), -1), (dict(bt=None), -1), (dict(lens=None), -1), (dict(pool=A + 8), -3),
    (dict(codes=A + 8), -3), (dict(scales=A + 4), -3),
])
def test_c_read_refusals(change, rc):
    a = dict(pool=A, pb=4, dst=A, codes=A, scales=A, bt=A, mb=4, lens=A, B=3, n_kv=2, d=64, bs=16,
             nb=2, fmt=K.VMPS_CACHE_E4M3, dtype=1, stream=None)
    a.update(change)
    assert _lib().vmps_read_cache8(*a.values()) == rc


def test_c_signatures_take_every_argument():
    lib = _lib()
    for name, n in (("vmps_norm_rope_and_cache", 25), ("vmps_read_cache8", 16),
                    ("vmps_paged_decode_attention_cache8", 20)):
        assert len(getattr(lib, name).argtypes) == n
        assert getattr(lib, name).restype is ctypes.c_int


def test_argument_structs_match_the_header(tmp_path):
    """Each field lies where the packed form puts it (compiled from include/vmps.h)."""
    import re
    import shutil
    import struct
    import subprocess

    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "vmps.h")
    text = open(header).read()
    structs = {"vmps_norm_rope_args": K._STORE_ARGS, "vmps_read_args": K._READ_ARGS,
               "vmps_decode_cache8_args": K._DECODE_ARGS}
    lines, want = [], []
    for name, packed in structs.items():
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        fields = [f.replace("*", " ").split()[-1] for d in body.split(";") for f in d.split(",") if f.strip()]
        codes = [c for n, c in re.findall(r"(\d*)([PqNfi])", packed.format) for _ in range(int(n or 1))]
        assert len(fields) == len(codes)
        at = 0
        for f, c in zip(fields, codes):
            size = struct.calcsize("@" + c)
            at = -(-at // size) * size
            want.append((name, f, at, size))
            at += size
            lines.append(f'printf("%zu %zu\\n", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));')
    src = tmp_path / "f.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(void) {%s return 0;}\n'
                   % (header, "\n".join(lines)))
    subprocess.run([shutil.which("gcc") or "cc", "-o", str(tmp_path / "f"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "f")], check=True, capture_output=True, text=True).stdout.split("\n")
    for (name, f, at, size), line in zip(want, got):
        assert line == f"{at} {size}", (name, f)


def test_null_argument_structs_are_refused():
    lib = _lib()
    for name in ("vmps_norm_rope_and_cache_args", "vmps_read_cache8_args",
                 "vmps_paged_decode_attention_cache8_args"):
        assert getattr(lib, name)(None, None) == -1
