"""The runtime provisions private memory per hardware queue for a full device -- frame x 64 lanes x 32 wave slots x 256 compute units, one block F -- out of 32 GiB for all queues
of a process.  Two queues fit whatever they run and wherever the other one's block lies (it leaves two holes, the larger one of at least (32 GiB - F) / 2) as long as 3 F <= 32 GiB,
that is, as long as no kernel's frame exceeds 21 845 bytes."""
import importlib
import os
import sys

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
sys.path.insert(0, os.path.join(ROOT, "tools"))
SLOTS = 32 * 256


def test_two_queues_fit_whatever_kernel_they_run(tmp_path):
    import check_long_branch as clb
    import kernel_resources as kr
    b = importlib.import_module("ps-signature-and-el-passo_amd.build")
    frames = {}
    for co in clb.extract_code_objects(b.build_hip(), str(tmp_path)):
        frames.update({k: int(v["private_segment_fixed_size"]) for k, v in kr.kernel_fields(co).items()})
    assert len(frames) > 60 and max(frames.values()) > 13000      # the verification kernels are among them
    too_big = {k: v for k, v in frames.items() if 3 * v * 64 * SLOTS > 32 << 30}
    assert too_big == {}
