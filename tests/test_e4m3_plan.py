"""The plan of the 8-bit decode attention as seen from the host: the scratch that sizes want."""
import subprocess
import sys
import threading

from util import ROOT

SIZES = [(B, 8, nkv, hd, hd, keys) for B in (1, 7, 64) for nkv in (1, 4) for hd in (64, 128, 256)
         for keys in (1000, 5000, 131072)]


def first_calls():
    """16 threads whose first calls of the library are made at the same time."""
    from agave_b200 import kernels
    f = kernels.library().agv_attention_decode_e4m3_scratch
    gate, got = threading.Barrier(16), [None] * 16

    def ask(i):
        gate.wait()
        got[i] = [f(*s) for s in SIZES]
    threads = [threading.Thread(target=ask, args=(i,)) for i in range(16)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(g == got[0] for g in got) and min(got[0]) >= 0 < max(got[0])


def test_first_calls_of_many_threads_agree():
    """The number of multiprocessors is asked for on the first call of a device."""
    code = "import sys; sys.path[:0] = ['.', 'tests']; import test_e4m3_plan as t; t.first_calls()"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_scratch_grows_with_the_keys():
    """Past the point where stretches begin, too."""
    from agave_b200 import kernels
    f = kernels.library().agv_attention_decode_e4m3_scratch
    for B, nh, nkv, hd, hdv, _ in SIZES:
        wants = [f(B, nh, nkv, hd, hdv, k) for k in (1, 1024, 4096, 16384, 65536, 1 << 20, (1 << 31) - 1)]
        assert wants == sorted(wants), (B, nkv, hd, wants)
