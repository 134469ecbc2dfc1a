"""Calls on 4-bit KV caches without a GPU: the refusals of the library's host code against a pretended HIP runtime, and the numpy form
that the GPU tests compare with."""
import os
import subprocess

import numpy as np
import pytest

import kv_q4_ref as R
from conftest import ROOT


def run_host(name, tmp_path):
    """tests/host/<name>.cpp, linked with the library and the pretended runtime, ends with 0."""
    here, lib, exe = os.path.join(ROOT, "tests", "host"), os.path.join(ROOT, "wick_amd", "lib", "libwick_rocm.a"), str(tmp_path / name)
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(here, name + ".cpp"),
           os.path.join(here, "fake_hip.cpp"), lib, "-lpthread", "-o", exe]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


def test_calls_that_are_refused(tmp_path):
    here, lib, exe = os.path.join(ROOT, "tests", "host"), os.path.join(ROOT, "wick_amd", "lib", "libwick_rocm.a"), str(tmp_path / "kv_q4_calls")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(here, "kv_q4_calls.cpp"),
           os.path.join(here, "fake_hip.cpp"), lib, "-lpthread", "-o", exe]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


def test_what_splits_and_shares_leave_fits_the_scratch(tmp_path):
    run_host("kv_q4_scratch", tmp_path)


def test_attention_over_no_row_asks_for_heads_too(tmp_path):
    run_host("kv_q4_no_rows", tmp_path)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_a_value_is_off_by_half_a_step_and_the_scale(hd):
    """|x - held| <= d / 2 where the rounding is, d where the largest step is cut off (15 for 16), both with the scale's rounding (2^-11 of up to 8
    steps) and that of the f32 steps."""
    x = np.random.default_rng(hd).standard_normal((50, 3, hd)).astype(np.float32)
    c = R.Cache(64, 3, hd)
    c.append(5, x)
    d = np.abs(c.scales[:, 5:55].astype(np.float64)).repeat(32, -1)
    off = np.abs(c.values(5, 50) - x.transpose(1, 0, 2)) / d
    top = x.reshape(50, 3, -1, 32).transpose(1, 0, 2, 3)
    cut = (c.words[:, 5:55, :, None] >> R.SHIFTS & np.uint32(15)).reshape(off.shape) == 15
    assert np.all(off[~cut] <= 0.5 + 8 * 2.0 ** -11 + 1e-5) and np.all(off[cut] <= 1 + 8 * 2.0 ** -11 + 1e-5)
    assert np.all(np.abs(top).max(-1) <= 8 * (1 + 2.0 ** -10) * np.abs(c.scales[:, 5:55].astype(np.float64)))
    assert np.isnan(c.values(0, 5)).all() and np.isnan(c.values(55, 9)).all()


def test_weights_of_the_numpy_form_add_up():
    k, v = R.Cache(40, 2, 64), R.Cache(40, 2, 64)
    x = np.random.default_rng(1).standard_normal((2, 40, 2, 64)).astype(np.float32)
    k.append(0, x[0]), v.append(0, x[1])
    _, p = R.attention(np.ones((10, 6, 64)), k, v, 30)
    assert np.allclose(R.gathered(p, 2).sum(1), 30) and not p[:, 0, 31:].any()


def test_ties_leave_the_higher_rows():
    assert R.evicted(np.array([5, 1, 1, np.nan, 1, 0, 9.0]), 7, 1, 1, 3).tolist() == [0, 2, 4, 6]
