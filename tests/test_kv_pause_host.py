"""Calls on a paged key/value cache while the process is paused, on the host stand-in of the HIP calls: those that name tracked memory are
refused, the others run."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "host_standin"))


def test_only_tracked_memory_is_refused_while_paused(tmp_path):
    import build_kv_standin
    lib = build_kv_standin.build(tmp_path)
    r = subprocess.run([sys.executable, os.path.join(HERE, "kv_pause_worker.py"), lib], env=dict(os.environ, AMEM_ENABLE="1", GMM_LOG="0"),
                       cwd=os.path.dirname(HERE), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert "kv pause worker: all done" in r.stdout
