"""CPU: the refusals of the MLA attention entry points (moe_kv_host.h compiled
here, no GPU), the rotary frequencies against the oracle's, and the 8-bit row
format's own reference against its definition."""
import os
import subprocess

import numpy as np
import pytest

import mla_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GOOD = {"cache", "no_seqs", "rope", "rope_in_place", "rope_head_major", "rope_nothing", "rope_broadcast_in", "no_scaling",
        "write", "write_bare", "read", "query"}


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("kv") / "kv_checks")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(ROOT, "tests", "kv_checks.cc"), "-o", exe],
                   check=True)
    return subprocess.run([exe], capture_output=True, text=True, timeout=60, check=True).stdout.splitlines()


def test_refusals(said):
    got = dict(line.split(": ", 1) for line in said if ": " in line)
    assert len(got) >= 60
    assert {k for k, v in got.items() if v == "ok"} == GOOD


def test_rotary_frequencies(said, oracle):
    turns = np.array([float(line.split()[2]) for line in said if line.startswith("turn ")])
    want = R.freqs()
    assert np.allclose(turns * 2 * np.pi, want, rtol=1e-14)
    # the reference's own formula in fp32: powf, a division and the blend, a few roundings of 2^-24
    cfg = oracle.mla_cfg()
    ref = np.array([oracle.lib().or_yarn_freq(__import__("ctypes").byref(cfg), i) for i in range(32)])
    assert np.allclose(want, ref, rtol=16 * 2.0 ** -24)


def test_null_context_is_refused(cuda_lib):
    from flash_deepseek_b200 import _lib
    lib = _lib.load()
    c, b, r, q = _lib.KVCacheC(), _lib.KVBatchC(), _lib.RopeConfigC(), _lib.MlaQueryC()
    assert lib.moe_rope_device(None, r, None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, 0, None) == -1
    assert lib.moe_kv_write_device(None, c, b, None, 0, 0, None, 0.0, None, None, None) == -1
    assert lib.moe_kv_read_device(None, c, b, None, 0, 0, None) == -1
    assert lib.moe_mla_attention_device(None, c, b, q, None, 0, None) == -1
    assert lib.moe_mla_workspace_bytes(None, 512) == 0


def test_row_bytes(cuda_lib):
    for fmt in R.FORMATS:
        for latent in (128, 256, 384, 512):
            assert cuda_lib.kv_row_bytes(fmt, latent) == R.row_bytes(fmt, latent)
    assert cuda_lib.kv_row_bytes(R.F16, 64) == 0 and cuda_lib.kv_row_bytes(7, 512) == 0


def test_quantize_reference():
    """The 8-bit reference keeps half a step, and its scale is the least one that fits."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((64, 128)) * 10.0 ** rng.integers(-4, 4, (64, 1))).astype(np.float32).astype(np.float64)
    x[0, :32] = 0
    x[1, 5] = 448.0
    x[1, :5] = x[1, 6:32] = 1.0
    codes, sb = R.quantize(x)
    k = sb.astype(int) - 127
    sc = np.repeat(2.0 ** k, 32, 1)
    err = np.abs(E(codes) * sc - x)
    step = np.maximum(np.abs(x) / 16, sc * 2.0 ** -10)
    fits = np.repeat(np.max(np.abs(x).reshape(64, 4, 32), -1) <= 448 * 2.0 ** k, 32, 1)
    assert np.all((err <= step) | ~fits) and np.all(k[~fits.reshape(64, 4, 32)[..., 0]] == 7)
    assert k[1, 0] == 0 and np.all(codes[0, :32] == 0) and k[0, 0] == -15


def E(codes):
    return R.E4M3[codes]


def test_work_division(tmp_path):
    exe = str(tmp_path / "kv_plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-unknown-pragmas", os.path.join(ROOT, "tests", "kv_plan.cc"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout
    cut, whole = int(r.stdout.split()[1]), int(r.stdout.split()[3])
    assert cut > 1000 and whole > 1000
