"""Static checks of the gfx950 listings of the kernels as they are shipped: compiled with the flags that the Makefile compiles them with, as register
allocation, spills and the choice of instructions depend on them."""
import concurrent.futures
import functools
import os
import re
import subprocess
import sys
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "adt_str_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")

# (file, kernels it must see at least): every translation unit with inline-asm loads or LDS reads and waits of its own
SOURCES = [("htsat_fused", 20), ("gemm", 30), ("gemm_i8", 30), ("kv4", 10), ("attention", 5), ("attention_fwd", 4), ("attention_bwd_fused", 3), ("attention_bwd_fused8", 2),
           ("htsat", 10)]


@functools.lru_cache(maxsize=None)
def flags():
    out = subprocess.run(["make", "-s", "--no-print-directory", "-C", CSRC, "print-cxxflags"], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    return tuple(out.stdout.split())


def compiled(name):
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, name + ".s")
        out = subprocess.run([HIPCC, *flags(), "-S", "--cuda-device-only", "-o", path, os.path.join(CSRC, name + ".hip")], cwd=d, capture_output=True, text=True, timeout=900)
        assert out.returncode == 0, out.stderr[-2000:]
        with open(path) as f:
            return f.read()


@pytest.fixture(scope="module")
def listings():
    flags()
    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        return dict(zip((n for n, _ in SOURCES), pool.map(compiled, (n for n, _ in SOURCES))))


def test_packed_fp32_is_off_where_kernels_are_compiled():
    assert "-packed-fp32-ops" in flags()
    with open(os.path.join(ROOT, "tools", "build_variant.sh")) as f:
        assert "print-cxxflags" in f.read()                     # variants of a kernel are built with the same flags


@pytest.mark.parametrize("name,min_kernels", SOURCES)
def test_no_register_is_touched_with_an_lds_read_pending_and_no_packed_fp32(listings, tmp_path, name, min_kernels):
    text = listings[name]
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    path = tmp_path / f"{name}.s"
    path.write_text(text)
    chk = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "probe", "check_pending_lds_regs.py"), str(path)], capture_output=True, text=True)
    assert chk.returncode == 0, chk.stdout[-4000:]
    assert chk.stdout.count(" 0 instruction(s)") >= min_kernels, chk.stdout[-2000:]


def scratch_bytes(text):
    """Kernel -> bytes of scratch per lane, from the listing's metadata."""
    kernels = re.findall(r"^\s+\.name:\s+(\S+)$(.*?)^\s+\.private_segment_fixed_size:\s+(\d+)$", text, re.M | re.S)
    return {name: int(size) for name, between, size in kernels if ".name:" not in between}


def test_the_training_and_serving_kernels_keep_their_registers(listings):
    """An accumulator array that is indexed at run time goes to memory whole: 528 bytes a lane in the 256 x 256 products, once a compiler limit kept their
    last loop rolled.  A few dwords are spills of addresses."""
    for name, min_kernels in SOURCES:
        sizes = scratch_bytes(listings[name])
        assert len(sizes) >= min_kernels, name
        for kernel, size in sizes.items():
            if "gemm_bf16_kernel" in kernel:                    # the fallback for operands that the others do not take
                continue
            most = 0 if name in ("gemm", "gemm_i8", "kv4") else 32
            assert size <= most, (kernel, size)
