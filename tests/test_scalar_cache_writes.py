"""Nothing here writes memory through the scalar data cache: neither the sources (hand-written, generated, generators, measurement
programs), nor the machine code of the built libraries.  Such a write is not coherent with the vector path, and machines that refuse
it refuse the whole tree for one mention.  What needs a wave-uniform fetch-and-add (the claims of the dynamic 8192-point loop) takes
a returning vector atomic of one lane; its wait discipline in the emulator is tested here too."""
import os
import re
import subprocess
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools", "gen"))

# (put together from parts: this file is one of the sources that are searched)
WRITES = re.compile(r"\bs_(?:buffer_|scratch_)?(?:%s)[_a-z]|\bs_dcache_(?:%s)" % ("|".join(("ato" + "mic", "sto" + "re")), "|".join(("w" + "b", "disc" + "ard"))))
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def test_the_pattern_knows_the_instructions():
    for part in (("s_", "atomic_add s92, s[90:91], 0x0 glc"), ("s_", "store_dword s0, s[2:3], 0x0"), ("s_buffer_", "store_dword s0"),
                 ("s_scratch_", "store_dword s0"), ("s_buffer_", "atomic_add s0"), ("s_dcache_", "wb"), ("s_dcache_", "discard s[0:1], 0")):
        assert WRITES.search("".join(part)), part
    for t in ("global_atomic_add v97, v104, v97, s[90:91] sc0", "s_load_dword s0, s[2:3], 0x0", "s_dcache_inv", "__hip_atomic_store (p, 0u)",
              "ds_write_b64 v0, v[2:3]", "global_store_dwordx2 v0, v[2:3], s[0:1]", "launch_ola_s_atoms"):
        assert not WRITES.search(t), t


def test_no_source_names_a_write_through_the_scalar_cache():
    hits = []
    for top, dirs, files in os.walk(ROOT):
        dirs[:] = [d for d in dirs if d not in (".git", "__pycache__", ".pytest_cache", "gpurun_out", "_work", "build", "lib")]
        for f in files:
            if f.endswith((".hip", ".h", ".hpp", ".inc", ".c", ".cc", ".cpp", ".s", ".S", ".asm", ".ll", ".py", ".sh", ".mk", ".cmake")) or f == "Makefile":
                p = os.path.join(top, f)
                for n, line in enumerate(open(p, errors="replace"), 1):
                    if WRITES.search(line):
                        hits.append("%s:%d: %s" % (os.path.relpath(p, ROOT), n, line.strip()[:80]))
    assert hits == []


@pytest.mark.parametrize("lib", ["libprot_hip.so", "libprot_hip_hooks.so"])
def test_no_built_library_holds_one(lib, tmp_path):
    """the device code of the libraries built here (a stale one would still hold what the sources no longer do)"""
    src = os.path.join(ROOT, "phaserotate.lv2_amd", "lib", lib)
    if not os.path.exists(src) or not os.path.exists(OBJDUMP):
        pytest.skip("library or llvm-objdump not there")
    (tmp_path / lib).write_bytes(open(src, "rb").read())
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    objs = sorted(p for p in os.listdir(tmp_path) if p.endswith("gfx950"))
    assert objs
    n_ins, claims = 0, 0
    for o in objs:
        txt = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", o], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        bad = [line.strip() for line in txt.splitlines() if WRITES.search(line)]
        assert bad == [], (o, bad[:4])
        n_ins += txt.count("\n")
        claims += len(re.findall(r"\bglobal_atomic_add\b.*\bsc0\b", txt))
    assert n_ins > 50000 and claims > 0


def _one_draw(wait, off=0):
    """lane 0 adds 1 to a word and the old value becomes wave-uniform, with or without the wait between the two"""
    from isa import Prog, Emu, V, S, SP, Lit
    P = Prog()
    P.auto = False
    P.v_mov(V(1), Lit(off))
    P.v_mov(V(0), Lit(1))
    P.exec_lane0()
    P.global_atomic_add(V(0), V(1), V(0), SP(10))
    P.exec_all()
    if wait:
        P.s_wait_vm_here(0)
    P.v_readfirstlane(S(20), V(0))
    emu = Emu(lds_bytes=256, n_threads=64)
    ctr = np.array([7, 40], np.uint32)
    emu.map(0x1000, ctr)
    emu.s[:, 10], emu.s[:, 11] = 0x1000, 0
    emu.run(P)
    return int(emu.s[0, 20]), ctr.tolist(), emu.v[0]


@pytest.mark.parametrize("off,old,after", [(0, 7, [8, 40]), (4, 40, [7, 41])])
def test_emulated_draw_is_one_lane_and_has_to_be_waited_for(off, old, after):
    got, ctr, v = _one_draw(True, off)
    assert got == old and ctr == after and (v[1:] == 1).all()      # (one add, the other lanes keep what they held)
    with pytest.raises(RuntimeError, match="in flight"):
        _one_draw(False, off)
    with pytest.raises(RuntimeError, match="unmapped"):
        _one_draw(True, 4096)


@pytest.mark.parametrize("hs,mode", [(8, 0), (12, 2), (13, 0)])
def test_a_dynamic_loop_that_does_not_wait_for_its_ticket_is_caught(hs, mode):
    """the draw moved behind the output stores: the counted wait at the top of the loop then no longer covers it, and the emulator
    says so (the planted mistake lives here, on the CPU, only)"""
    import gen_olasave8k as G8

    class Late(G8.Gen8kDyn):
        def claim_issue(self):
            if self.loop_reached:
                return                     # (the loop's own draw is made in epilogue_row below)
            super().claim_issue()

        def epilogue_row(self, u, k):
            super().epilogue_row(u, k)
            if k == self.HS - 1:
                super().claim_issue()

        def loop(self):
            self.loop_reached = True
            super().loop()

        loop_reached = False

    G8.self_test_dyn(hs, mode, nb=2, xr=0, stride=1, verbose=False)
    keep = G8.Gen8kDyn
    G8.Gen8kDyn = Late
    try:
        with pytest.raises(RuntimeError, match="in flight"):
            G8.self_test_dyn(hs, mode, nb=2, xr=0, stride=1, verbose=False)
    finally:
        G8.Gen8kDyn = keep
