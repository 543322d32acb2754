"""The C++ layers around the experts without a GPU: host_block_layers.cpp against the C ABI compiled for the host, whose launchers are stand-ins."""
import os
import subprocess

from tests.conftest import ROOT


def test_layers_and_refusals(tmp_path):
    csrc, exe = os.path.join(ROOT, "omega-ai_amd", "csrc"), str(tmp_path / "layers")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-w", "-D__HIP_PLATFORM_AMD__", "-D__align__(n)=__attribute__((aligned(n)))", "-DHIP_SYMBOL(x)=((const void *)(x))",
                           "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), "-I" + csrc,
                           "-I" + os.path.join(ROOT, "omega-ai_amd", "host"), "-o", exe, "-x", "c++"]
                          + [os.path.join(csrc, f) for f in ("api.hip", "ops_api.hip", "block_api.hip")]
                          + [os.path.join(ROOT, "tests", f) for f in ("host_runtime.cpp", "host_ops.cpp", "host_block.cpp", "host_block_layers.cpp")])
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.endswith("0 failed\n"), got.stdout + got.stderr
