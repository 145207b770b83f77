"""CPU: rotary frequencies away from the default configuration, against the
oracle (pinned to the reference engine's own functions) and the 64-bit form."""
import ctypes as C
import os
import subprocess

import numpy as np

import mla_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# dim, theta, scale, orig_ctx, beta_fast, beta_slow: other bases, scales and lengths; a context that passes the longest
# wavelength (the ramp's end stays at the last pair); one shorter than the shortest (the whole ramp in front); betas
# that cross; small and large dims
CASES = [(64, 500000, 8, 8192, 32, 1), (64, 10000, 4, 2048, 32, 1), (64, 10000, 40, 100000, 32, 1), (64, 10000, 16, 6, 32, 1),
         (128, 1000000, 2, 32768, 32, 1), (80, 10000, 40, 4096, 16, 2), (64, 10000, 40, 4096, 1, 32), (2, 10000, 8, 4096, 32, 1),
         (256, 150.5, 3.5, 777, 32, 1), (64, 10000, 1, 4096, 32, 1)]


def table(tmp_path):
    exe = str(tmp_path / "kv_ramp")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(ROOT, "tests", "kv_ramp.cc"), "-o", exe], check=True)
    said = subprocess.run([exe], input="".join(" ".join(map(str, c)) + "\n" for c in CASES), capture_output=True, text=True,
                          timeout=60, check=True).stdout
    return [np.array(line.split(), float) * 2 * np.pi for line in said.splitlines()]


def test_frequencies_of_other_configurations(tmp_path, oracle):
    got = table(tmp_path)
    assert len(got) == len(CASES)
    pinned = 0
    for f, (dim, theta, scale, orig, fast, slow) in zip(got, CASES):
        want = R.freqs(dim, theta, scale, orig, fast, slow)
        assert len(f) == dim // 2 and np.allclose(f, want, rtol=1e-13)
        if (fast, slow) != (32, 1) or scale == 1:
            continue   # the reference has these betas built in
        cfg = oracle.mla_cfg(qk_rope=dim, rope_theta=theta, rope_scale=scale, rope_orig_ctx=orig)
        ref = np.array([oracle.lib().or_yarn_freq(C.byref(cfg), i) for i in range(dim // 2)])
        # fp32: a power (2 ulp of an exponent up to 7 in log2 theta), a division, the ramp, a blend
        assert np.allclose(f, ref, rtol=32 * 2.0 ** -24)
        pinned += 1
    assert pinned >= 6


def test_last_pair_of_a_context_past_every_wavelength(tmp_path):
    """The ramp ends at the last pair, which is divided by the whole scale."""
    f = table(tmp_path)[2]
    plain = 10000.0 ** (-np.arange(32) / 32)
    assert np.isclose(f[31] * 40, plain[31], rtol=1e-12) and f[0] == 1.0 and f[31] < f[30] < plain[30]
