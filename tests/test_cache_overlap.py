"""Caches whose rows share memory are refused before a kernel could race on them; layouts that only
share an allocation are not.  The C entry decides, so this runs on the CPU with pointers that are no
addresses: a call that is not refused fails at its launch there."""

import pytest
import torch

OK_BUT_NO_DEVICE, REFUSED = 3, 1
BASE = 1 << 20


def cache_write(k, v, ks=None, vs=None, B=2, cap=8, H=2, D=64, T=3, ct=3):
    """k, v, ks, vs: (byte offset, sb, st, sh) of the caches and their scales."""
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would start a kernel")
    from multiscreen import _native
    L = _native.lib()
    c = [(BASE + x[0], *x[1:]) if x is not None else (0, 0, 0, 0) for x in (k, v, ks, vs)]
    row = (BASE << 8, T * H * D, H * D, D)
    rc = L.msa_cache_write(_native.pack_cache_args(*row, *row, *c[0], *c[1], *c[2], *c[3], 0, 0, 0, 0, 0, B, T, T, H, D, 1, cap, ct),
                           None)
    if rc == REFUSED:
        assert "share memory" in L.msa_last_error().decode()
    return rc


HEAD = (1024, 64, 512)     # head-major codes of 2 x 8 x 2 rows of 64 bytes
SC = (16, 1, 8)            # their scales
FAR = 1 << 16              # bytes


def write(k=(0, *HEAD), v=(FAR, *HEAD), ks=(2 * FAR, *SC), vs=(3 * FAR, *SC), **kw):
    return cache_write(k, v, ks, vs, **kw)


def test_rows_of_their_own_are_taken():
    assert write() == OK_BUT_NO_DEVICE
    # (B, T, H, D) order; slices of longer storage; one sequence, head or position with any stride
    assert write(k=(0, 1024, 128, 64), v=(FAR, 1024, 128, 64)) == OK_BUT_NO_DEVICE
    assert write(k=(0, 4096, 64, 2048), v=(1024, 4096, 64, 2048)) == OK_BUT_NO_DEVICE
    assert write(k=(0, 0, 64, 512), v=(FAR, 16, 64, 512), ks=(2 * FAR, 0, 1, 8), vs=(3 * FAR, 0, 1, 8), B=1) == OK_BUT_NO_DEVICE
    # k and v side by side: rows, heads, sequences
    assert write(k=(0, 2048, 128, 1024), v=(64, 2048, 128, 1024)) == OK_BUT_NO_DEVICE
    assert write(k=(0, 2048, 64, 512), v=(1024, 2048, 64, 512)) == OK_BUT_NO_DEVICE
    assert write(k=(0, *HEAD), v=(2048, *HEAD)) == OK_BUT_NO_DEVICE
    # rows of codes with their scale behind them (80 bytes), k and v in one row (160 bytes)
    assert write(k=(0, 1280, 80, 640), ks=(64, 320, 20, 160)) == OK_BUT_NO_DEVICE
    assert write(k=(0, 2560, 160, 1280), ks=(64, 640, 40, 320), v=(80, 2560, 160, 1280), vs=(144, 640, 40, 320)) == OK_BUT_NO_DEVICE
    # a head's codes, then its scales
    assert write(k=(0, 1152, 64, 576), ks=(512, 288, 1, 144)) == OK_BUT_NO_DEVICE
    # 16-bit rows of the model's type
    assert cache_write((0, *HEAD), (2 * FAR, *HEAD), ct=1) == OK_BUT_NO_DEVICE


def test_shared_rows_are_refused():
    for kw in (dict(v=(0, *HEAD)),                                        # kcache is vcache
               dict(vs=(2 * FAR, *SC)),                                   # one tensor of scales for both
               dict(v=(64, *HEAD)), dict(v=(1024, *HEAD)),                # shifted by a position, by a sequence
               dict(v=(1024 + 512 + 7 * 64, *HEAD)),                      # the last row alone
               dict(k=(0, 1024, 32, 512)), dict(k=(0, 512, 64, 512)),     # rows, sequences that overlap
               dict(k=(0, 1024, 64, 448)), dict(ks=(2 * FAR, 16, 1, 7)),  # heads that do
               dict(k=(0, 960, 64, 512)),
               dict(ks=(64, *SC)), dict(ks=(FAR + 4, *SC)),               # scales among the codes of either
               dict(k=(0, 1280, 80, 640), ks=(60, 320, 20, 160)),
               dict(v=(16, 2048, 64, 512), k=(0, *HEAD))):                # different layouts over one range
        assert write(**kw) == REFUSED, kw
    assert cache_write((0, *HEAD), (FAR, *HEAD), ct=1) == OK_BUT_NO_DEVICE
    assert cache_write((0, *HEAD), (2048, *HEAD), ct=1) == REFUSED        # 16-bit rows reach twice as far
    big = 1 << 62                                                         # strides whose products leave 64 bits
    far = dict(ks=(2 * FAR, big // 4, 1, 8), vs=(3 * FAR, big // 4, 1, 8))
    assert write(k=(0, big, 64, 512), v=(0, big, 64, 512), **far) == REFUSED
    assert write(k=(0, big, 64, 512), v=(FAR, big, 64, 512), **far) == OK_BUT_NO_DEVICE


def test_a_read_does_not_write_rows_twice():
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would start a kernel")
    from multiscreen import _native
    L = _native.lib()

    def read(k, v):
        c = [(BASE + 4 * FAR + i * FAR, *HEAD) for i in (0, 1)] + [(BASE + 6 * FAR + i * FAR, *SC) for i in (0, 1)]
        return L.msa_cache_read(_native.pack_cache_args(BASE + k[0], *k[1:], BASE + v[0], *v[1:], *c[0], *c[1], *c[2], *c[3], 0, 0, 0,
                                                        0, 0, 2, 3, 3, 2, 64, 1, 8, 3), None)

    row = (384, 128, 64)
    assert read((0, *row), (FAR, *row)) == OK_BUT_NO_DEVICE
    assert read((0, *row), (0, *row)) == REFUSED and "share memory" in L.msa_last_error().decode()
    assert read((0, 192, 64, 64), (FAR, *row)) == REFUSED
    # the cache itself may be an expanded one
    c = (BASE + 4 * FAR, 0, 64, 512)
    s = (BASE + 6 * FAR, 0, 1, 8)
    assert L.msa_cache_read(_native.pack_cache_args(BASE, *row, BASE + FAR, *row, *c, *c, *s, *s, 0, 0, 0, 0, 0, 2, 3, 3, 2, 64, 1, 8, 3),
                            None) == OK_BUT_NO_DEVICE
