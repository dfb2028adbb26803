"""Calls of the attention that are refused before anything is launched, and the calls beside them that are not."""
import ctypes
import random

import pytest
import torch

from sarathi_serve_b200 import _native as N

without_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="makes calls on addresses that are not device memory")


def shape(heads=8, kv=2, hd=128, page=16, dtype=2, window=0, requests=4, tokens=64):
    return N.AttentionShape(heads, kv, hd, page, dtype, window, requests, tokens)


def attention(s, **k):
    """Status of a call on made-up addresses, far from each other unless told otherwise."""
    lib, sp = N.lib(), ctypes.byref(s)
    x = dict(out=1 << 34, ldo=1024, lse=None, q=1 << 35, ldq=1280, T=8, cache=1 << 36, pages=10, scale=0.1)
    x.update(k)
    return lib.sb200_paged_attention(x["out"], x["ldo"], x["lse"], x["q"], x["ldq"], x["T"], x["cache"], x["pages"], 4096, sp, 4096, 10,
                                     x["scale"], 0, 1 << 40, lib.sb200_attention_workspace_bytes(sp), None, None)


def said(rc, what):
    return rc == 1 and what in N.lib().sb200_last_error()


@without_gpu
def test_lse_on_top_of_another_array():
    """8 rows of 1024 elements of 2 bytes in out (1280 apart in the second half) and q, lse 8 x 8 x 4 = 256 bytes."""
    s = shape()
    out, q, cache = 1 << 34, 1 << 35, 1 << 36
    page = 2 * 16 * 2 * 128 * 2
    for lse in (out, out - 252, out + 8 * 2048 - 4, out + 5000, q, q - 4, q + 7 * 2560, q + 3 * 2560 + 2044, q + 2560 - 128, cache + 64,
                cache + 10 * page - 4, cache - 200):
        assert said(attention(s, lse=lse), b"lse must not overlap"), hex(lse)
    for lse in (out - 256, out + 8 * 2048, q - 256, q + 7 * 2560 + 2048, q + 2048, q + 4 * 2560 + 2048 + 256, cache - 256, cache + 10 * page):
        assert not said(attention(s, lse=lse), b"overlap"), hex(lse)
    assert said(attention(s, lse=out + 2560 * 2, ldo=1280), b"lse must not overlap")
    assert not said(attention(s, lse=out + 2560 * 2 + 2048, ldo=1280), b"overlap")


@without_gpu
def test_lse_between_rows_as_found_by_trying_them_all():
    s = shape()
    rng = random.Random(1)
    out = 1 << 34
    for _ in range(2000):
        T, ldo = rng.randint(1, 12), 1024 + 8 * rng.choice([0, 1, 15, 16, 17, 40, 200])
        lse = out + 4 * rng.randint(-200, T * ldo // 2 + 200)
        meet = any(lse < out + i * ldo * 2 + 2048 and out + i * ldo * 2 < lse + T * 32 for i in range(T))
        assert said(attention(s, T=T, ldo=ldo, lse=lse), b"lse must not overlap") == meet, (T, ldo, lse - out)


@without_gpu
def test_rows_too_far_apart():
    """Offsets of q rows are kept in 32 bits, in units of 16 bytes: 64 GiB, which a strided view of a large buffer can pass."""
    for dtype, es in ((2, 2), (0, 4)):
        s = shape(dtype=dtype, tokens=1 << 20)
        T = 1 << 20
        far = ((1 << 32) - 1) * 16 // es // T // 8 * 8
        assert not said(attention(s, T=T, ldq=far, q=1 << 50), b"too far apart")
        assert said(attention(s, T=T, ldq=far + 8, q=1 << 50), b"too far apart")
        assert said(attention(s, T=2, ldq=1 << 62, q=1 << 50), b"too far apart")
        assert said(attention(s, T=8, ldo=1 << 61), b"too far apart")
