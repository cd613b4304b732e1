"""Packed fp32 instructions (v_pk_add_f32, v_pk_mul_f32, v_pk_fma_f32) stay out of the device code: some of their forms can give wrong results without an error.  The compiler makes
them from ordinary float code unless its target feature is off, so the built code itself is looked at, and every recipe that compiles device code."""
import os
import re
import shutil
import subprocess

from genefaceplusplus_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def test_no_packed_fp32_in_the_library(tmp_path):
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.check_call([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, stdout=subprocess.DEVNULL)
    images = sorted(f for f in os.listdir(tmp_path) if "gfx950" in f)
    assert images
    mfma = 0
    for image in images:
        code = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", image], cwd=tmp_path, capture_output=True, text=True, check=True).stdout
        mfma += code.count("v_mfma_")
        assert not re.search(r"v_pk_(add|mul|fma)_f32", code), image
    assert mfma > 1000                   # (the code was there to be read)


def test_every_device_compile_keeps_them_out():
    for folder in ("genefaceplusplus_amd", "tools", "oracle"):
        for base, _, files in os.walk(os.path.join(ROOT, folder)):
            for name in files:
                if name != "Makefile" and not name.endswith((".py", ".sh", ".md", ".hip")):
                    continue
                path = os.path.join(base, name)
                text = open(path, encoding="utf-8", errors="replace").read()
                compiles = re.findall(r"--offload-arch(?:(?!--offload-arch)[\s\S])*", text)
                compiles = [c for c in compiles if not re.match(r"\S+ *,? *\"?-shared", c.replace('"', ""))]         # (a link has no device code to make)
                for c in compiles:
                    assert "-packed-fp32-ops" in c or ("NO_PACKED_F32" in c and "-packed-fp32-ops" in text), (path, c[:120])
