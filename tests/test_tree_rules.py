"""What the tree must not hold, shown on the sources alone: each test reads the files under version control (or, where git is absent, every file of the same folders) and names
the lines at fault.  The scans are textual, so a pattern here is spelled in a way that does not match itself."""
import os
import re
import subprocess

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
SOURCE_SUFFIXES = (".py", ".sh", ".js", ".h", ".hip", ".cc", ".cpp", ".c", ".s", "Makefile")


def source_files():
    """Repository-relative paths of the sources, scripts and build files."""
    r = subprocess.run(["git", "-C", ROOT, "ls-files", "-z"], capture_output=True, text=True)
    if r.returncode == 0:
        names = [n for n in r.stdout.split("\0") if n]
    else:
        names = []
        for top in ("include", "oracle", "ps-signature-and-el-passo_amd", "tests", "tools"):
            for dp, _, fs in os.walk(os.path.join(ROOT, top)):
                names += [os.path.relpath(os.path.join(dp, f), ROOT) for f in fs]
        names += [f for f in os.listdir(ROOT) if os.path.isfile(os.path.join(ROOT, f))]
    return sorted(n for n in names if n.endswith(SOURCE_SUFFIXES) and os.path.exists(os.path.join(ROOT, n)))


def hits(pattern):
    rx = re.compile(pattern)
    out = []
    for n in source_files():
        with open(os.path.join(ROOT, n), errors="replace") as f:
            out += ["%s:%d: %s" % (n, i, ln.strip()) for i, ln in enumerate(f, 1) if rx.search(ln)]
    return out


def test_the_scan_sees_the_sources():
    """An empty list of files would make every test below pass."""
    names = source_files()
    assert "bench.py" in names and "ps-signature-and-el-passo_amd/csrc/elp/pipeline.h" in names and "oracle/Makefile" in names


def test_no_build_switch_ends_a_verification_early_and_no_script_reproduces_a_fault():
    """A verification that returns before its last step accepts what it did not check, so no compile-time switch of that kind stays in the device headers; and a GPU fault whose
    cause is known is guarded on the CPU (test_isa_hazards.py), never made to happen again by a script."""
    assert hits(r"ELP_[B]ISECT") == []
    assert [n for n in source_files() if re.search(r"fault_(repro|probe)", n)] == []
    assert hits(r"[_]fault_(repro|probe)\b") == []


def test_nothing_runs_searches_or_patches_a_prebuilt_module():
    """Vectors come from source built here or from data already recorded; no script loads the reference's prebuilt modules, reads their memory image or writes into it, and no
    text calls the BLS12-381 vectors an ordinary run of the reference."""
    assert hits(r"[w]asm-build|HEAP[U](8|16|32)\b|select[C]urve|wasm[_](curve|verify)") == []
    assert [n for n in source_files() if n.endswith(".js")] == []
    claim = re.compile(r"wasm run on (this|that|the) curve|run on BOTH curves|reference-run oracle|BLS12-381 is pinned|pinned (on|by) (BOTH|both) curves|both curves by (proofs|reference)", re.I)
    texts = source_files() + ["README.md", "DESIGN.md", "INTEGRATION.md"]
    assert [n for n in texts if n != "tests/test_tree_rules.py" and claim.search(open(os.path.join(ROOT, n), errors="replace").read())] == []


def test_no_source_names_a_write_through_the_scalar_data_cache():
    """GPU code writes through vector stores only, and the tree says so to a reader of its text: no source, script or build file names a scalar store, a scalar atomic, or the
    write-back and discard of that cache."""
    assert hits(r"\bs_(buffer_|scratch_)?(store|atomic)_|\bs_d""cache_(wb|discard)") == []


def test_long_branch_scanner_accepts_only_saves_that_a_compiled_function_makes(tmp_path):
    """The return address counts as saved by a lane write or a copy into other scalar registers, before the first clobbering s_getpc_b64; anything else in that place -- a vector
    store of unrelated registers, a scalar one of s[30:31] -- leaves the function reported."""
    import sys
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import check_long_branch as clb
    body = "\tv_add_u32_e32 v0, v1, v2\n" * 4
    far = "\ts_getpc_b64 s[30:31]\n.Lpost_getpc1:\n\ts_add_u32 s30, s30, 12\n\ts_addc_u32 s31, s31, 0\n\ts_setpc_b64 s[30:31]\n"
    listing = "".join(name + ":\n" + before + body + far + body + "\ts_setpc_b64 s[30:31]\n" for name, before in (
        ("saved_in_lanes", "\tv_writelane_b32 v40, s30, 0\n\tv_writelane_b32 v40, s31, 1\n"), ("saved_as_pair", "\ts_mov_b64 s[34:35], s[30:31]\n"),
        ("saved_in_halves", "\ts_mov_b32 s34, s30\n\ts_mov_b32 s35, s31\n"), ("vector_store", "\tscratch_store_dword off, v40, s33\n"),
        ("scalar_store", "\ts_" + "store_dwordx2 s[30:31], s[4:5], 0x0\n")))
    p = tmp_path / "listing.s"
    p.write_text(listing)
    assert [b[0] for b in clb.scan(str(p))] == ["vector_store", "scalar_store"]


def test_every_stream_has_the_default_priority():
    """Streams of different priorities are not mixed: no stream, process group or graph asks for one."""
    assert hits(r"\bpriority\s*=|high_[p]riority|Stream\w*With[P]riority") == []
