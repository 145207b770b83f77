"""CPU: the work division of the MLA attention at the limits of its numbers, and buffers that it must not share."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_lengths_near_two_to_the_31(tmp_path):
    """A context length near 2^31 under a page table that long: the sequence is cut and reported, the others keep
    their shares."""
    exe = str(tmp_path / "kv_limits")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-unknown-pragmas", "-fsanitize=signed-integer-overflow",
                    "-fno-sanitize-recover", os.path.join(ROOT, "tests", "kv_limits.cc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok 450\n", r.stdout + r.stderr


def test_the_search_for_a_share_is_bounded():
    """The thread that finds the share's first sequence looks at its own stretch of sequences only."""
    text = open(os.path.join(ROOT, "flash_deepseek_b200", "csrc", "moe_mla.cu")).read()
    assert "for (;; b++)" not in text and re.search(r"for \(; b < b1 - 1; b\+\+\)", text)


def test_output_in_the_querys_place_is_refused(tmp_path):
    exe = str(tmp_path / "kv_in_place")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(ROOT, "tests", "kv_in_place.cc"), "-o", exe],
                   check=True)
    said = subprocess.run([exe], capture_output=True, text=True, timeout=60, check=True).stdout.splitlines()
    got = dict(line.split(": ", 1) for line in said)
    assert len(got) == 5 and {k for k, v in got.items() if v != "ok"} == {"latent", "rope"}
    api = open(os.path.join(ROOT, "flash_deepseek_b200", "csrc", "moe_api.cu")).read()
    assert "kv_bad_in_place(b, q)" in api[api.index("int moe_mla_attention_device"):]
