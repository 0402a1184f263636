"""What the entries of the 8-bit cache, the shared prefix and the token log probabilities refuse,
before any launch and without a device."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from orator_amd import _lib

FAKE = 0x1000  # never dereferenced: every call below is refused first
OK, INVALID, UNSUPPORTED, CAPACITY = (_lib.ORATOR_OK, _lib.ORATOR_ERR_INVALID,
                                      _lib.ORATOR_ERR_UNSUPPORTED, _lib.ORATOR_ERR_CAPACITY)


def rc(name, args, **change):
    vals = dict(args, **change)
    return getattr(_lib.lib(), "orator_" + name)(*vals.values())


WRITE = dict(k=FAKE, v=FAKE, stride=1024, kq=FAKE, ks=FAKE, vq=FAKE, vs=FAKE, Tq=4, Hkv=8, Dh=128,
             pos=FAKE, cap=64, stream=None)
WRITE_PAGED = dict(k=FAKE, v=FAKE, stride=1024, kq=FAKE, ks=FAKE, vq=FAKE, vs=FAKE, table=FAKE,
                   max_pages=4, ps=16, n_pages=8, B=2, Tq=4, Hkv=8, Dh=128, pos=FAKE, stream=None)
READ = dict(kq=FAKE, ks=FAKE, vq=FAKE, vs=FAKE, k=FAKE, v=FAKE, bf16=0, Tq=4, Hkv=8, Dh=128,
            pos=FAKE, cap=64, stream=None)
READ_PAGED = dict(kq=FAKE, ks=FAKE, vq=FAKE, vs=FAKE, table=FAKE, max_pages=4, ps=16, n_pages=8,
                  k=FAKE, v=FAKE, bf16=1, B=2, Tq=4, Hkv=8, Dh=128, pos=FAKE, stream=None)
DECODE = dict(q=FAKE, kq=FAKE, ks=FAKE, vq=FAKE, vs=FAKE, out=FAKE, Hq=16, Hkv=8, Dh=128, pos=FAKE,
              cap=64, scale=0.1, stream=None)
DECODE_PAGED = dict(q=FAKE, kq=FAKE, ks=FAKE, vq=FAKE, vs=FAKE, table=FAKE, max_pages=4, ps=16,
                    n_pages=8, pos=FAKE, out=FAKE, B=2, Hq=16, Hkv=8, Dh=128, scale=0.1, stream=None)
SHARED = dict(q=FAKE, kpool=FAKE, vpool=FAKE, table=FAKE, max_pages=4, ps=16, n_pages=8, pos=FAKE,
              shared=20, out=FAKE, B=2, Hq=16, Hkv=8, Dh=128, scale=0.1, stream=None)
SHARED_Q8 = dict(q=FAKE, kq=FAKE, ks=FAKE, vq=FAKE, vs=FAKE, table=FAKE, max_pages=4, ps=16,
                 n_pages=8, pos=FAKE, shared=20, out=FAKE, B=2, Hq=16, Hkv=8, Dh=128, scale=0.1,
                 stream=None)
LOGPROBS = dict(x=FAKE, stride=1000, tokens=FAKE, rows=3, vocab=1000, k=5, lp=FAKE, ent=FAKE,
                ids=FAKE, top=FAKE, stream=None)

ATTENTION = [("gqa_decode_q8", DECODE), ("gqa_decode_q8_paged", DECODE_PAGED),
             ("gqa_decode_shared_paged", SHARED), ("gqa_decode_shared_q8_paged", SHARED_Q8)]
CACHE = [("kv_write_q8", WRITE), ("kv_write_q8_paged", WRITE_PAGED), ("kv_read_q8", READ),
         ("kv_read_q8_paged", READ_PAGED)]


@pytest.mark.parametrize("name,args", ATTENTION + CACHE)
def test_sizes_of_zero_are_no_calls(name, args):
    for size in ("B", "Tq", "Hq", "Hkv", "Dh"):
        if size in args:
            for n in (0, -3):
                none = {k: None for k, v in args.items() if v == FAKE}
                assert rc(name, args, **{**none, size: n}) == OK


@pytest.mark.parametrize("name,args", ATTENTION + CACHE)
def test_null_pointers_and_misaligned_caches(name, args):
    for k in (k for k, v in args.items() if v == FAKE):
        assert rc(name, args, **{k: None}) == INVALID, k
        assert b"null" in _lib.lib().orator_last_error()
    for k in ("kq", "ks", "vq", "vs", "kpool", "vpool"):
        if k in args:
            assert rc(name, args, **{k: FAKE + 8}) == INVALID, k


@pytest.mark.parametrize("name,args", ATTENTION + CACHE)
def test_shapes(name, args):
    for dh in (8, 24, 100, 272, 1024):
        change = dict(Dh=dh)
        if "stride" in args:
            change["stride"] = 8 * dh
        assert rc(name, args, **change) == UNSUPPORTED
    if "ps" in args:
        for ps in (0, -16, 8, 24, 48):
            assert rc(name, args, ps=ps) == INVALID
        for n in ("max_pages", "n_pages"):
            assert rc(name, args, **{n: 0}) == INVALID
            assert rc(name, args, **{n: -1}) == INVALID
    else:
        for cap in (0, -16, 8, 40, 0x7fffffff):
            assert rc(name, args, cap=cap) == INVALID
    if "Hq" in args:
        assert rc(name, args, Hq=12) == INVALID
        assert rc(name, args, Hq=65536) == UNSUPPORTED
        if "B" in args:
            assert rc(name, args, B=65536) == UNSUPPORTED
    if "shared" in args:
        assert rc(name, args, shared=-1) == INVALID
        assert rc(name, args, shared=65) == CAPACITY
    if "stride" in args:
        assert rc(name, args, stride=1023) == INVALID
    if "bf16" in args:
        assert rc(name, args, bf16=2) == INVALID


@pytest.mark.parametrize("name,args", ATTENTION + CACHE)
@pytest.mark.parametrize("dh", [16, 64])
def test_more_rows_than_a_grid_holds(name, args, dh):
    """Sizes that are ints each, but 2^24 workgroups or more together."""
    if "Tq" in args:
        for tq, hkv in ((1 << 30, 8), (1 << 25, 1), (1, 1 << 25), (0x7fffffff, 0x7fffffff)):
            if dh == 64 and hkv == 1 and tq == 1 << 25:
                tq <<= 4  # blocks of 16 rows
            assert rc(name, args, Tq=tq, Hkv=hkv, Dh=dh, **(
                {"stride": hkv * dh} if "stride" in args else {})) == UNSUPPORTED
            assert b"too many" in _lib.lib().orator_last_error()
    elif "B" in args:
        assert rc(name, args, B=65535, Hq=65534, Hkv=2, Dh=dh) == UNSUPPORTED
        assert rc(name, args, B=1 << 15, Hq=1 << 9, Hkv=1, Dh=dh) == UNSUPPORTED


def test_token_logprobs():
    for n in ("rows", "vocab"):
        assert rc("token_logprobs", LOGPROBS, **{n: 0}) == OK
    assert rc("token_logprobs", LOGPROBS, lp=None, ent=None, ids=None, top=None) == OK
    assert rc("token_logprobs", LOGPROBS, x=None) == INVALID
    assert rc("token_logprobs", LOGPROBS, tokens=None) == INVALID
    assert rc("token_logprobs", LOGPROBS, stride=999) == INVALID
    assert rc("token_logprobs", LOGPROBS, ids=None) == INVALID
    assert rc("token_logprobs", LOGPROBS, top=None) == INVALID
    for k in (-1, 33):
        assert rc("token_logprobs", LOGPROBS, k=k) == UNSUPPORTED
    assert rc("token_logprobs", LOGPROBS, vocab=4, k=5) == UNSUPPORTED


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_blocks_of_captured_graphs(tmp_path):
    """The workspace's bookkeeping of blocks that belong to one capture (tests/cpp)."""
    src = Path(__file__).resolve().parent / "cpp" / "test_workspace_capture.cc"
    exe = tmp_path / "test_workspace_capture"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-pthread", "-fsanitize=address,undefined",
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    assert "workspace capture OK" in out.stdout
