"""The key/value cache in 8 bits without a GPU: the argument checks of the C ABI, and the rounding that its kernels use, for every pair of a value and a magnitude."""
import os
import subprocess

import numpy as np
import pytest
import torch

from oracle import kv_cache as ok

N = None
S = (64, 64, 64, 1)


def test_refusals_of_the_c_abi():
    from cpm_kernels_amd.library import cpmk

    def write(b=1, h=1, n=4, d=64, length=64, block=16, k=16, pos_each=N, pos=0, keys=16):
        cpmk.kv_write_int8(b, h, n, d, length, block, k, *S, k, *S, pos_each, pos, N, keys, keys, keys, keys, N)

    def read(b=1, h=1, n=4, d=64, length=64, block=16, k=16, keys=16):
        cpmk.kv_read_int8(b, h, n, d, length, block, keys, keys, keys, keys, N, 0, k, k, *S, N)

    def attend(b=1, h=2, kv=1, n=4, d=64, length=64, block=16, q=16, keys=16, lens_each=N, len=8, bias=N, mapping=N, buckets=32, distances=128, both=0, space=16):
        cpmk.kv_attention_int8(b, h, kv, n, d, length, block, q, *S, keys, keys, keys, keys, lens_each, len, N, -1, 1, 0.125, bias, mapping, buckets,
                               distances, both, N, 0, 0, q, *S, space, N)
    for call in (write, read, attend):
        for bad in (dict(b=-1), dict(n=-1), dict(block=48), dict(block=0), dict(keys=N), dict(length=-64)):
            with pytest.raises(RuntimeError, match="invalid argument"):
                call(**bad)
        for bad in (dict(d=72), dict(length=72), dict(keys=24)):
            with pytest.raises(RuntimeError, match="divisibility"):
                call(**bad)
        for bad in (dict(d=272), dict(length=2 ** 25)):
            with pytest.raises(RuntimeError, match="limit"):
                call(**bad)
        with pytest.raises(RuntimeError, match="invalid argument"):         # (a cache without positions)
            call(length=0, **(dict(len=0) if call is attend else {}))
        for empty in (dict(b=0, keys=N), dict(n=0, keys=N), dict(d=0, keys=N)):
            call(**empty)
    for bad in (dict(k=N), dict(pos=-1), dict(pos=61), dict(pos=2 ** 31 - 1)):
        with pytest.raises(RuntimeError, match="invalid argument"):
            write(**bad)
    for bad in (dict(q=N), dict(kv=0), dict(h=3, kv=2), dict(len=-1), dict(len=65), dict(bias=16), dict(bias=16, mapping=16, buckets=0),
                dict(bias=16, mapping=16, distances=0), dict(length=0, len=0)):
        with pytest.raises(RuntimeError, match="invalid argument"):
            attend(**bad)
    for bad in (dict(bias=16, mapping=16, distances=1025), dict(bias=16, mapping=16, distances=513, both=1), dict(n=2 ** 30, h=2)):
        with pytest.raises(RuntimeError, match="limit"):
            attend(**bad)
    assert cpmk.kv_attention_int8_workspace(0, 4, 4, 1, 64, 64) == 0 and cpmk.kv_attention_int8_workspace(1, 4, 3, 1, 64, 64) == 0


def test_refusals_of_sizes_whose_products_leave_64_bits():
    """A product of sizes that comes round to 0 is neither an empty call nor a small grid."""
    from cpm_kernels_amd.library import cpmk
    big = 2 ** 30

    def refused(call, *args):
        with pytest.raises(RuntimeError, match="limit"):
            call(*args)
    p = 16
    refused(cpmk.kv_attention_int8, 2 ** 18, 2 ** 18, 2 ** 18, 2 ** 20, 256, 64, 16, p, *S, p, p, p, p, N, 8, N, -1, 1, 0.125, N, N, 0, 0, 0, N, 0, 0, p, *S, p, N)
    refused(cpmk.kv_attention_int8, big, big, big, 16, 64, 64, 16, p, *S, p, p, p, p, N, 8, N, -1, 1, 0.125, N, N, 0, 0, 0, N, 0, 0, p, *S, p, N)
    for tokens in (1, 2048, 4096):
        refused(cpmk.kv_write_int8, big, big, tokens, 64, 4096, 16, p, *S, p, *S, N, 0, N, p, p, p, p, N)
        refused(cpmk.kv_read_int8, big, big, tokens, 64, 4096, 16, p, p, p, p, N, 0, p, p, *S, N)
    assert cpmk.kv_attention_int8_workspace(big, big, big, 16, 64, 64) == 0
    assert cpmk.kv_attention_int8_workspace(2 ** 18, 2 ** 18, 2 ** 18, 2 ** 20, 256, 64) == 0
    # (no work is no work whatever the other sizes are)
    cpmk.kv_attention_int8(big, big, big, 0, 64, 64, 16, N, *S, N, N, N, N, N, 8, N, -1, 1, 0.125, N, N, 0, 0, 0, N, 0, 0, N, *S, N, N)
    cpmk.kv_write_int8(big, big, 0, 64, 4096, 16, N, *S, N, *S, N, 0, N, N, N, N, N, N)


def test_positions_and_lengths_that_are_no_integers():
    """They are refused, not cut off; integers of any kind are taken."""
    from cpm_kernels_amd.torch.kv_cache import _each
    here = torch.device("cpu")
    for x in (5, np.int32(5), np.int64(5), 5.0):
        assert _each(x, 2, here) == (None, 5)
    for x in (5.5, -0.25, float("nan"), float("inf"), None, "5", torch.tensor(5), torch.tensor([5, 5]), torch.tensor([5, 5, 5], dtype=torch.int32)):
        with pytest.raises((AssertionError, TypeError, ValueError, OverflowError)):
            _each(x, 2, here)


def test_oracle_of_the_cache():
    """Ties away from zero, older integers rounded again, what lies behind a write untouched."""
    ints, top = np.full((1, 1, 32, 16), 9, np.int8), np.zeros((1, 1, 2), np.float16)
    x = np.zeros((1, 1, 2, 16), np.float16)
    x[0, 0, 0, :5] = [127, 63.5, -63.5, 0.5, 0.25]
    ok.write(ints, top, x, [3], [1])
    assert ints[0, 0, 3, :5].tolist() == [127, 64, -64, 1, 0] and top[0, 0].tolist() == [127, 0]
    assert (ints[0, 0, :3] == 0).all() and (ints[0, 0, 4:] == 9).all()          # (older tokens beside an old magnitude of 0)
    x[0, 0, 0, :2] = [254, np.nan]
    ok.write(ints, top, x, [4], [1])
    assert ints[0, 0, 3, :5].tolist() == [64, 32, -32, 1, 0] and ints[0, 0, 4, :2].tolist() == [127, 0] and top[0, 0, 0] == 254
    v = np.arange(2 * 32 * 48).reshape(1, 2, 32, 48).astype(np.int8)
    assert np.array_equal(ok.by_token(ok.by_sixteen(v)), v) and ok.by_sixteen(v)[0, 1, 1, 40, 5] == v[0, 1, 21, 40]


def test_rounding_of_every_pair(tmp_path):
    here = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "kv_round_check.c")
    exe = str(tmp_path / "kv_round_check")
    subprocess.run(["gcc", "-O2", "-ffp-contract=off", "-fopenmp", here, "-o", exe, "-lm"], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    assert "0 differ" in out, out


def test_rounding_of_every_pair_as_the_kernels_compile_it(tmp_path):
    """The functions of csrc/kv_round.h themselves, a fused product and addition: what rounds is not left to a compiler's choice.  The factors are divisions rounded as IEEE says on both sides."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "kv_round_fma_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-fopenmp", "-I", os.path.join(root, "cpm_kernels_amd", "csrc"),
                    os.path.join(root, "tests", "native", "kv_round_fma_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    assert out.splitlines()[-1] == "0 differ", out
