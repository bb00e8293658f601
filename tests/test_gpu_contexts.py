"""Several contexts on one device.  The runtime provisions private memory per hardware queue, for a full device whatever the grid: frame x 64 lanes x 32 wave slots x compute
units, 8 GiB for the 16 KB frames of the largest kernels.  Contexts that each launch on a queue of their own use up the space there is for it (four queues), and the next dispatch
that needs a larger block aborts its queue.  So the contexts of a device launch on ONE stream."""
import importlib
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))

CHILD = r"""
import ctypes, importlib, re, sys
sys.path.insert(0, %r)
elp = importlib.import_module("ps-signature-and-el-passo_amd")
synth = importlib.import_module("ps-signature-and-el-passo_amd.synth")

def run(ctx):
    wl = synth.Workload(ctx, 8, seed=83, window_bits=8)
    recs, mask, expect = wl.verify_id_batch(64, 4, with_retrieval=True)
    flags, accepted, held = ctx.verify_id_batch_aggregated(recs, mask, True, wl.ad, bytes(range(32)))
    assert held and (flags == expect).all() and accepted == int(expect.sum())

def used():
    path = next(m.group(1) for ln in open("/proc/self/maps") for m in [re.search(r"(\S*libamdhip64\S*)", ln)] if m)
    f, t = ctypes.c_size_t(), ctypes.c_size_t()
    assert ctypes.CDLL(path).hipMemGetInfo(ctypes.byref(f), ctypes.byref(t)) == 0
    return (t.value - f.value) / 2 ** 20

a, b = elp.Context(elp.CURVE_BN254, 0), elp.Context(elp.CURVE_BN254, 0)
run(a)
one = used()
run(b)
two = used()
run(a)                      # and back: both contexts go on giving the same answers
print("MIB", one, two, used(), flush=True)
a.close()
run(b)                      # the stream outlives the context that came first
b.close()
c = elp.Context(elp.CURVE_BN254, 0)      # ... and a later context gets one again
run(c)
c.close()
print("DONE", flush=True)
"""


def test_a_second_context_needs_no_second_block_of_private_memory():
    """In a process of its own (a fresh runtime): the second context's first aggregated verification adds its tables and workspaces (some tens of MiB), not 8 GiB."""
    r = subprocess.run([sys.executable, "-c", CHILD % ROOT], capture_output=True, text=True, timeout=100, cwd=ROOT,
                       env=dict(os.environ, GPU_MAX_HW_QUEUES="4"))          # HIP's own default: the streams of two contexts would land on two queues
    assert r.returncode == 0 and "DONE" in r.stdout, r.stdout + r.stderr
    one, two, three = (float(x) for x in r.stdout.split("MIB")[1].split()[:3])
    print("used after one context %.0f MiB, after two %.0f, after the first again %.0f" % (one, two, three))
    assert two - one < 1024 and three - two < 1024, (one, two, three)


def test_launch_stream_option_and_two_contexts_at_once(elp):
    """Two contexts in two threads on the shared stream, then on the two launch streams, then back: every verdict and count is the generator's.  Other values are refused and
    leave the context working."""
    import threading
    synth = importlib.import_module("ps-signature-and-el-passo_amd.synth")
    ctxs = [elp.Context(elp.CURVE_BN254, 0) for _ in range(2)]
    try:
        loads = []
        for i, c in enumerate(ctxs):
            wl = synth.Workload(c, 8, seed=89 + i, window_bits=8)
            loads.append((wl, wl.verify_id_batch(700 + i, 4, with_retrieval=True, corrupt_every=9, corrupt_at=4)))
        for which in (0, 1, 0):
            ctxs[1].set_launch_stream(which)
            for bad in (-1, 2):
                with pytest.raises(elp.ElpassoError):
                    ctxs[1].set_launch_stream(bad)
            got = [[], []]

            def work(i):
                wl, (recs, mask, _) = loads[i]
                for _ in range(3):
                    got[i].append(ctxs[i].verify_id_batch(recs, mask, True, wl.ad))

            threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            for i in range(2):
                expect = loads[i][1][2]
                assert len(got[i]) == 3 and all((fl == expect).all() and cnt == int(expect.sum()) for fl, cnt in got[i]), (which, i)
    finally:
        for c in ctxs:
            c.close()
