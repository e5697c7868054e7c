"""CPU: lanes of a wave that exchange values through LDS without a workgroup barrier need a fence of the wave between the
writes and the reads, and between those reads and the next writes: without one the compiler, which orders only what a
thread's own addresses make it, may move them across each other.  Read off the LLVM code of the device compilation."""
import importlib
import os
import re
import subprocess

import pytest

build = importlib.import_module("gaussian-splatting_amd.build")


def _device_code(source):
    """{kernel: its LDS events in the order of the text}: "S" store, "L" load, "F" fence of the wave or barrier."""
    path = os.path.join(build.CSRC, source)
    r = subprocess.run([build.HIPCC, *build.COMMON, *build.SOURCES[source], "--cuda-device-only", "-emit-llvm", "-S", "-o", "-", path],
                       stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    kernels, events = {}, None
    for line in r.stdout.splitlines():
        m = re.match(r"define .*amdgpu_kernel void @(\w+)", line)
        if m:
            events = kernels.setdefault(m.group(1), [])
        elif line == "}":
            events = None
        elif events is not None:
            if re.search(r"amdgcn\.(wave|s)\.barrier\(", line):
                events.append("F")
            elif re.match(r"\s+store .* addrspace\(3\)|.* @llvm\.memcpy\.p3\.", line):
                events.append("S")
            elif re.match(r"\s+%\S+ = load .* addrspace\(3\)|.* @llvm\.memcpy\.p\d+\.p3\.", line):
                events.append("L")
    return {k: re.sub(r"(.)\1+", r"\1", "".join(e)) for k, e in kernels.items()}


def test_rows_of_packed_sh_leave_between_fences():
    found = {k: e for k, e in _device_code("sh_pack.hip").items() if "S" in e}
    assert len(found) == 1 + 1 + 8                       # quantise; dequantise; gradients of four degrees, few and several views
    for kernel, events in found.items():
        assert "SL" not in events and "LS" not in events, (kernel, events)


def test_view_records_leave_between_fences():
    found = {k: e for k, e in _device_code("preprocess.hip").items() if "S" in e}
    assert len(found) == 8                               # records: fast and general, packed or not, opacities per view or not
    for kernel, events in found.items():
        assert "SL" not in events and "LS" not in events, (kernel, events)
        assert events.startswith("F"), (kernel, events)  # the loop over the views comes back to the stores


def test_parameter_gradients_leave_behind_a_fence():
    found = {k: e for k, e in _device_code("param_bwd.hip").items() if "S" in e}
    assert len(found) == 8
    for kernel, events in found.items():                 # in front: a thread's own column, written and read by itself alone
        assert re.fullmatch(r"(SL)+SFL", events), (kernel, events)
