"""Rows that overlap: the check behind the paged-cache operators' refusals against a byte map, and the refusals of the C
entries (their pointers are never touched)."""
import os
import shutil
import subprocess

import pytest

from strataflow_b200 import lib as L

from test_paged_ops import APPEND, DECODE, PREFILL, X, call, sfk  # noqa: F401 (sfk: a fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_meet(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "paged_rows_check")
    subprocess.run([gxx, "-std=c++17", "-O1", "-I", os.path.join(ROOT, "strataflow_b200", "csrc"),
                    os.path.join(ROOT, "tests", "paged_rows_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


ROW = 8 * 64 * 4  # bytes of a token's q


@pytest.mark.parametrize("kw", [
    dict(qs=8 * 64 + 8),                       # out of a wider q: sequence 1's output lies in sequence 0's gap and row 1
    dict(out=X + 4), dict(out=X + ROW), dict(out=X - ROW), dict(out=X + 2 * ROW), dict(out=X - 2 * ROW),
    dict(qs=3 * 8 * 64, out=X + 2 * ROW),      # behind row 0, reaching row 1
    dict(n=1, out=X + ROW - 4), dict(n=1, out=X - ROW + 4),
])
def test_decode_refuses_an_out_that_overlaps_q(sfk, kw):  # noqa: F811
    assert call(sfk, "sfk_attn_decode_window", DECODE, **kw) == L.SFK_ERR_INVALID_ARGUMENT
    assert b"overlaps q" in sfk.sfk_last_error()


@pytest.mark.parametrize("kw", [
    dict(), dict(qs=12 * 64), dict(out=X + 4), dict(out=X + ROW), dict(out=X - 4 * ROW), dict(out=X + 4 * ROW),
    dict(n_tok=1), dict(qs=6 * 8 * 64, out=X + 2 * ROW),
])
def test_prefill_refuses_an_out_that_overlaps_q(sfk, kw):  # noqa: F811
    assert call(sfk, "sfk_attn_prefill_window", PREFILL, **kw) == L.SFK_ERR_INVALID_ARGUMENT
    assert b"overlaps it" in sfk.sfk_last_error()


@pytest.mark.parametrize("kw,why", [
    (dict(outs=8 * 64 + 8), b"overlaps q"), (dict(out=X + 4), b"overlaps q"), (dict(out=X + ROW), b"overlaps q"),
    (dict(out=X - 3 * ROW + 4, outs=8 * 64), b"overlaps q"), (dict(qs=12 * 64, outs=8 * 64), b"overlaps q"),
    (dict(k=X + ROW - 4, v=X + (1 << 16)), b"overlaps k or v"),
    (dict(k=X + (1 << 16), v=X + 2 * ROW, vs=4 * 64), b"overlaps k or v"),
    (dict(n=1, k=X + ROW - 4, v=X + (1 << 16)), b"overlaps k or v"),
])
def test_append_refuses_a_q_out_that_overlaps_other_rows(sfk, kw, why):  # noqa: F811
    kw = {"k": X + (1 << 16), "v": X + (1 << 17), **kw}
    assert call(sfk, "sfk_qk_norm_rope_append", APPEND, **kw) == L.SFK_ERR_INVALID_ARGUMENT
    assert why in sfk.sfk_last_error()
