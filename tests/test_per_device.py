"""What the launching code remembers of a device is kept for each: ``csrc/per_device.h`` compiled for the host against a runtime with several devices, and the files that go by it."""
import os
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "mini_trainer_b200" / "csrc"
CUDA_INC = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"

MAIN = r"""
#include "per_device.h"
#include <stdio.h>
static int current = 0, asked = 0;
static bool broken = false;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = current; return broken ? cudaErrorInitializationError : cudaSuccess; }
extern "C" cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int d) { ++asked; *v = 100 + d; return cudaSuccess; }
extern "C" cudaError_t cudaGetLastError() { return cudaSuccess; }
static mtb::PerDevice<bool> configured;
static int sets = 0;
static void launch() { if (bool& done = configured.here(); !done) { ++sets; done = true; } }
int main() {
  int bad = 0;
  for (int round = 0; round < 2; ++round)
    for (current = 0; current < 64; ++current) { launch(); bad += mtb::sms_here() != 100 + current; }
  bad += sets != 64 || asked != 64;            // each device once
  for (current = 64; current < 66; ++current) for (int i = 0; i < 2; ++i) launch();   // beyond what is remembered: each time
  bad += sets != 68;
  current = 65;
  bad += mtb::sms_here() != 165;
  broken = true;
  launch();
  bad += sets != 69 || mtb::sms_here() != 148;
  broken = false; current = 3;
  launch();
  bad += sets != 69 || mtb::sms_here() != 103;
  printf("wrong %d\n", bad);
  return bad;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None or not (CUDA_INC / "cuda_runtime.h").exists(), reason="no host compiler or CUDA headers")
def test_each_device_has_its_own(tmp_path):
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = tmp_path / "per_device"
    build = subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(CUDA_INC), "-I", str(CSRC), "-o", str(exe), str(tmp_path / "main.cpp")], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout


@pytest.mark.parametrize("name", ["newton_schulz.cu", "route_balance.cu", "nll.cu", "gemm_tcgen05.cu", "gemm2_tcgen05.cu"])
def test_attributes_and_sizes_are_kept_by_device(name):
    """The operators that make their backend's device the current one, and the products they are made of: no kernel's attribute and no number of a device in a variable that all devices share."""
    text = (CSRC / name).read_text()
    for call in re.finditer(r"cudaFuncSetAttribute\(|cudaOccupancyMaxActiveClusters\(|cudaDeviceGetAttribute\(", text):
        start = text.rfind("\nstatic ", 0, call.start())
        assert "PerDevice<" in text[max(start, text.rfind("\ntemplate", 0, call.start())):call.start()], text[call.start() - 200:call.end()]
    assert not re.search(r"static (bool|int) (configured|\w*sms|known|pairs|n)\b", text)
