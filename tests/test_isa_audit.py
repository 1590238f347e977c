"""Static audit of the compiled gfx950 code (no GPU needed: hipcc cross-compiles to assembly).

The fused MLP kernels issue their LDS fragment reads by hand (inline asm) so that hipcc cannot sink them next
to their use; the price is that the compiler's s_waitcnt bookkeeping does not protect those registers.  The
audit (scripts/audit_asm_loads.py) walks the emitted ISA and fails if any instruction touches the destination
of a hand-issued read before a covering `s_waitcnt lgkmcnt`, or if compiler-generated code uses M0, which the
LDS-DMA pieces overwrite without restoring; scripts/audit_scratch.py then holds every kernel symbol to its scratch
allowance (csrc/scratch_allow.txt: zero for everything but two scalar-spill kernels).

`make -C torch-nerf_amd/csrc audit` is the one implementation of it (the same command __graft_entry__.build() runs): it
compiles the five audited translation units to assembly IN PARALLEL and only when a source changed (csrc/build/*.s), so a
warm tree answers in seconds and a cold one in the time of the largest unit instead of the sum of all five."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "torch-nerf_amd", "csrc")
AUDITED = ["mlp_forward", "mlp_backward", "mlp_forward_bf16", "render_fused", "mlp_layered"]


@pytest.fixture(scope="module")
def audit_output():
    out = subprocess.run(["make", "-C", CSRC, "-j8", "audit"], capture_output=True, text=True)
    assert out.returncode == 0, (out.stdout + out.stderr)[-3000:]
    return out.stdout


@pytest.mark.parametrize("name", AUDITED)
def test_hand_issued_reads_are_waited_for(audit_output, name):
    lines = [ln for ln in audit_output.splitlines() if ln.startswith(f"build/{name}.s:")]
    assert len(lines) == 1 and "hand-issued LDS reads, 0 problems" in lines[0], audit_output[-2000:]
    assert int(lines[0].rsplit(":", 1)[1].split()[0]) > 100      # the audit really saw the reads


def test_no_kernel_spills_beyond_its_allowance(audit_output):
    """A scratch reload is a VMEM load whose vmcnt wait also waits for the weight DMA: every kernel symbol is held to
    csrc/scratch_allow.txt (a file-wide allowance would hide a new spill in any of the layered family's ~50 instances)."""
    lines = [ln for ln in audit_output.splitlines() if ln.startswith("scratch audit:")]
    assert len(lines) == 1 and lines[0].endswith("0 over their allowance"), audit_output[-2000:]
    assert int(lines[0].split()[2]) >= 60                         # every kernel of the five files was looked at


def test_every_kernel_file_is_audited(audit_output):
    files = sorted(f[:-4] for f in os.listdir(CSRC) if f.endswith(".hip"))
    assert len(files) >= 17
    for name in files:
        assert f"build/{name}.s: " in audit_output, name


@pytest.mark.parametrize("line,bad", [("v_pk_fma_f32 v[0:1], v[2:3], v[4:5], v[0:1]", True), ("v_pk_mul_f32 v[0:1], v[2:3], s[4:5]", True),
                                      ("v_pk_add_f32 v[0:1], v[2:3], v[4:5] op_sel_hi:[1,0]", True),
                                      ("v_pk_add_f16 v0, v1, v2", False), ("v_fma_f32 v0, v1, v2, v3", False)])
def test_packed_fp32_instructions_fail_the_audit(tmp_path, line, bad):
    path = tmp_path / "k.s"
    path.write_text(f"_Z1kv:\n\ts_mov_b32 s0, 0\n\t{line}\n\ts_endpgm\n")
    out = subprocess.run(["python3", os.path.join(ROOT, "scripts", "audit_asm_loads.py"), str(path)], capture_output=True, text=True)
    assert out.returncode == int(bad) and ("packed fp32" in out.stdout) == bad, out.stdout + out.stderr


def test_a_variant_of_one_file_is_built_with_the_regular_flags(tmp_path):
    """scripts/variant_one_file.sh, with a compiler that only writes down its arguments: the flags of the regular build
    (`make -n`) and the extra define."""
    log, fake = tmp_path / "log", tmp_path / "hipcc"
    fake.write_text(f'#!/bin/bash\necho "$@" >> {log}\nwhile [ $# -gt 1 ]; do [ "$1" = -o ] && : > "$2"; shift; done\n')
    fake.chmod(0o755)
    name = f"test{os.getpid()}"
    made = [os.path.join(CSRC, f"build_{name}", "adam.hip.o"), os.path.join(CSRC, "..", "lib", "variants", f"{name}.so")]
    env = {**os.environ, "HIPCC": str(fake)}
    try:
        out = subprocess.run(["bash", os.path.join(ROOT, "scripts", "variant_one_file.sh"), name, "adam.hip", "-DX_TEST=1"],
                             env=env, capture_output=True, text=True)
        assert out.returncode == 0 and all(os.path.exists(m) for m in made), out.stdout + out.stderr
    finally:
        for m in made:
            if os.path.exists(m):
                os.remove(m)
        if os.path.isdir(os.path.dirname(made[0])):
            os.rmdir(os.path.dirname(made[0]))
    plain = subprocess.run(["make", "-C", CSRC, "-nB", "build/adam.hip.o"], env=env, capture_output=True, text=True).stdout
    regular = next(ln for ln in plain.splitlines() if " -c adam.hip" in ln).split(" -c ")[0].split()[1:]
    compiled, linked = log.read_text().splitlines()
    assert compiled.split(" -c ")[0].split() == regular + ["-DX_TEST=1"] and "-packed-fp32-ops" in regular
    assert "build/adam.hip.o" not in linked.split() and f"build_{name}/adam.hip.o" in linked
