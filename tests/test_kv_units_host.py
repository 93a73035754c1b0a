"""How attention over a paged key/value cache deals out its work, in host builds with sanitizers."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_driver(tmp_path, source):
    exe = str(tmp_path / "driver")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "asystem-amem_amd", "csrc"), os.path.join(ROOT, "tests", "kv_index", source), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "ok" in r.stdout


def test_units_of_any_offsets_stay_inside_the_tensors(tmp_path):
    run_driver(tmp_path, "unit_driver.cpp")


def test_cuts_with_the_kernels_own_figures(tmp_path):
    run_driver(tmp_path, "cut_rules_driver.cpp")
