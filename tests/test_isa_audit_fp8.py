"""The audit of the 8-bit products' counted waits on the compiler's listing, and that it finds what it is for: mistakes planted in the listing's text.
The build's check for register spills covers every source whose kernels count their waits, also where the kernel is in a header."""

import os
import re
import shutil

import pytest

import build
import isa_audit
from build import HIPCC

needs_hipcc = pytest.mark.skipif(shutil.which(HIPCC) is None, reason="needs hipcc")

KINDS = ["EPI_BF16, true", "EPI_GLU, true", "EPI_GLU_KEEP, true", "EPI_GLU_BWD_BF16, true", "EPI_GLU_BWD_F16, false", "EPI_F32, false"]


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    folder = tmp_path_factory.mktemp("isa_fp8")
    source, path = str(folder / "kinds.hip"), str(folder / "kinds.s")
    with open(source, "w") as f:
        f.write('#include "fp8_gemm.h"\nnamespace fmahip::fp8 {\n')
        for kind in KINDS:
            f.write(f"template __global__ void fp8_gemm_kernel<{kind}>(const GemmArgs);\n")
        f.write("}\n")
    isa_audit.compile_to_assembly(source, path)
    return path


@needs_hipcc
def test_counts(listing):
    assert len(list(isa_audit.kernels(listing, isa_audit.FP8_KERNEL))) == len(KINDS)
    assert isa_audit.audit_fp8(listing) == 0


@needs_hipcc
def test_finds_planted_mistakes(listing):
    """a counted wait that allows for one more, an operand load or a counted store left out, a scratch access"""
    for name, body in isa_audit.kernels(listing, isa_audit.FP8_KERNEL):
        assert not isa_audit.audit_fp8_kernel(name, body)
        epi = int(re.search(r"ILi(\d)E", name).group(1))
        stores, kind = isa_audit.FP8_STORES[epi]
        counted = {4, min(4 + stores, 62)}
        at = [(i, int(m.group(1))) for i, m in enumerate(re.search(r"vmcnt\((\d+)\)", s) for s in body) if m]
        after = lambda i: next(s for s in body[i + 1 :] if re.search(r"s_barrier|vmcnt|buffer_|global_|s_endpgm", s))  # noqa: E731
        waits = [i for i, n in at if n in counted and "s_barrier" in after(i)]
        assert waits
        for i in waits:
            more = re.sub(r"vmcnt\((\d+)\)", lambda m: f"vmcnt({int(m.group(1)) + 1})", body[i])
            assert isa_audit.audit_fp8_kernel(name, body[:i] + [more] + body[i + 1 :]), (name, body[i])
            loads = [j for j in range(i - 1, 0, -1) if body[j].strip().startswith("buffer_load_dwordx4") and " lds" in body[j]][:4]
            assert isa_audit.audit_fp8_kernel(name, body[: loads[-1]] + body[loads[-1] + 1 :]), name
        if kind:
            i = next(i for i, s in enumerate(body) if s.strip().startswith(kind))
            assert isa_audit.audit_fp8_kernel(name, body[:i] + body[i + 1 :]), name
        assert isa_audit.audit_fp8_kernel(name, body[:40] + ["\tscratch_load_dword v1, off, off"] + body[40:]), name


def test_scratch_is_refused_where_a_headers_kernel_counts_its_waits():
    csrc = os.path.join(os.path.dirname(build.__file__), "csrc")
    texts = {n: open(os.path.join(csrc, n)).read() for n in os.listdir(csrc)}
    found = set()
    for header, text in texts.items():
        counts = re.findall(r"(?:wait_vm<|waitcnt_imm\(\(int\)|vmcnt\()([^>)\n]+)", text)
        if header.endswith(".h") and any(c.strip() != "0" for c in counts):
            for kernel in re.findall(r"__global__[^;{]*?void (\w+)\(", text):
                for source in (n for n, t in texts.items() if n.endswith(".hip") and re.search(rf"\b{kernel}\s*<", t)):
                    found.add(source)
                    assert re.search(build.NO_SCRATCH_SOURCES[source], kernel), (source, kernel)
    assert {"fp8_gemm.hip", "grouped_gemm_ragged.hip", "grouped_gemm_ragged_tall.hip"} <= found
