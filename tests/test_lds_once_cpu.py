"""Kernels of more than 64 KB of LDS have that allowed on every device they run on, not on the first one alone."""
import ctypes as C
import glob
import os
import re
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "hexanima_amd", "csrc")


def test_each_device_once(tmp_path):
    so = str(tmp_path / "lds_once.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", so, os.path.join(HERE, "lds_once_host.cpp")], check=True)
    lib = C.CDLL(so)
    assert lib.host_allow(3, 1) == 7 and lib.host_sets() == 0  # what failed is tried again
    for dev in (3, 0, 3, 63, 0):
        assert lib.host_allow(dev, 0) == 0 and (lib.host_bytes(dev, 0), lib.host_bytes(dev, 1)) == (100, 200)
    assert lib.host_sets() == 6
    for _ in range(2):  # past the devices that are kept
        assert lib.host_allow(64, 0) == 0
    assert lib.host_sets() == 10


def test_no_launch_keeps_one_flag_for_all_devices():
    """hipFuncSetAttribute stands in lds_once.h and, with a list of devices, in causal_attn.h"""
    calls = {}
    for path in glob.glob(os.path.join(CSRC, "*.h*")):
        with open(path) as f:
            calls[os.path.basename(path)] = len(re.findall(r"hipFuncSetAttribute\(", f.read()))
    assert {n: k for n, k in calls.items() if k} == {"lds_once.h": 1, "causal_attn.h": 1}
