"""The compiled products of csrc/fp8_ops.hip and csrc/muon_ops.hip (gfx950 assembly, no GPU needed): what the
compiler does not look after for the loads into LDS that tile_product.h issues by inline assembly, and what no
kernel of theirs may hold."""
import os
import re
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "nerf-rep_for_test_amd")


@pytest.fixture(scope="module", params=["fp8_ops", "muon_ops", "experts_ops"])
def kernels(request, tmp_path_factory):
    """{kernel: its instructions in order} of one source, compiled with the library's flags."""
    out = str(tmp_path_factory.mktemp("isa") / (request.param + ".s"))
    flags = subprocess.check_output(["make", "-C", PKG, "-s", "--no-print-directory", "-f", "-", "flags"], text=True,
                                    input="include Makefile\nflags:\n\t@echo $(HIPFLAGS)\n").split()
    subprocess.check_call(["/opt/rocm/bin/hipcc", *flags, "-Wno-inline-asm", "--offload-device-only", "-S",
                           f"csrc/{request.param}.hip", "-o", out], cwd=PKG, stderr=subprocess.DEVNULL)
    found, name = {}, None
    for line in open(out):
        m = re.match(r"(_Z\w+):", line)
        if m:
            name = m.group(1)
            found[name] = []
        elif re.match(r"\s+[a-z]\w+", line) and name and not line.strip().startswith("."):
            found[name].append(line.split(";")[0].split("//")[0].strip())
        elif line.startswith("\t.end_amdhsa_kernel") or line.startswith(".Lfunc_end"):
            name = None
    return request.param, {k: v for k, v in found.items() if any(i.startswith("s_endpgm") for i in v)}


def regs(text):
    """{(file, number)} of the registers named in an operand list."""
    got = set()
    for f, a, b in re.findall(r"\b([sv])\[(\d+):(\d+)\]", text):
        got |= {(f, i) for i in range(int(a), int(b) + 1)}
    got |= {(f, int(a)) for f, a in re.findall(r"\b([sv])(\d+)\b", text)}
    return got


def test_scalar_operands_of_the_loads_into_lds_are_old_enough(kernels):
    """A scalar register that a vector instruction wrote may be read by a memory instruction 5 wait states later;
    m0 one after its write."""
    source, found = kernels
    loads = 0
    for name, code in found.items():
        for i, ins in enumerate(code):
            if not (ins.startswith("buffer_load") and ins.endswith("lds")):
                continue
            loads += 1
            scalars = {r for r in regs(ins) if r[0] == "s"}
            waits, j, m0 = 0, i - 1, None
            while j >= 0 and waits < 5:
                op = code[j].split()[0]
                if m0 is None and "m0" in code[j].split(",")[0] and op.startswith("s_mov"):
                    m0 = waits
                if op.startswith("v_"):
                    written = regs(code[j].split(",")[0])
                    assert not (written & scalars), (name, code[j], ins)
                waits += int(code[j].split()[1]) + 1 if op == "s_nop" else 1
                j -= 1
            assert m0 is not None and m0 >= 1, (name, code[max(0, i - 4):i + 1])
    assert loads > 0 if source != "experts_ops" else loads == 0


def test_no_packed_fp32_and_no_scratch_in_the_products(kernels):
    source, found = kernels
    assert found
    for name, code in found.items():
        assert not [i for i in code if re.match(r"v_pk_(add|mul|fma)_f32", i)], name
        if "product_kernel" in name:
            assert not [i for i in code if i.startswith("scratch_")], name
            assert sum(i.startswith("v_mfma") for i in code) >= 4, name


def test_a_step_waits_for_its_own_loads_only(kernels):
    """Between the barrier in a product's loop and its last matrix instruction there is no wait for memory."""
    source, found = kernels
    if source == "experts_ops":
        return
    for name, code in found.items():
        if "product_kernel" not in name:
            continue
        last = max(i for i, c in enumerate(code) if c.startswith("v_mfma"))
        first = max(i for i, c in enumerate(code[:last]) if c.startswith("s_barrier"))
        bad = [c for c in code[first:last] if c.startswith("s_waitcnt") and "vmcnt" in c]
        assert not bad, (name, bad)
