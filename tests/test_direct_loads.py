"""CPU: the direct loads into LDS that are written as inline assembly keep the wait states that the compiler does not count
into them, wherever their base was formed."""
import os
import subprocess

import pytest

from wekua_amd import build, check_main_loops

# Bases straight out of vector registers: each lane has an address, the first lane's is taken, and the load follows at once.
KERNEL = """
#include "wk_lds_dma.hpp"
using namespace wk::lds_dma;
__global__ void direct(const char *const *p, float *out, unsigned step) {
    __shared__ float lds[1024];
    const unsigned long long a = (unsigned long long)p[threadIdx.x];
    const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) float *)lds;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    %s((const void *)((unsigned long long)hi << 32 | lo), threadIdx.x * step, to);
    wait_vm<0>();
    out[threadIdx.x] = lds[threadIdx.x];
}
"""


@pytest.mark.parametrize("load", ["dma16", "dma4"])
def test_base_out_of_vector_registers(tmp_path, load):
    """Compiled, not run: no vector instruction may write the load's base within five wait states of it."""
    src, out = tmp_path / "direct.hip", tmp_path / "direct.s"
    src.write_text(KERNEL % load)
    flags = [f for f in build.HIP_FLAGS if f != "-fPIC"]
    subprocess.run([build.HIPCC] + flags + ["--cuda-device-only", "-S", str(src), "-o", str(out)], check=True, stdout=subprocess.DEVNULL,
                   stderr=subprocess.DEVNULL)
    text = out.read_text()
    assert "v_readfirstlane_b32" in text, "the case is not the one that is meant"
    loads, short = check_main_loops.short_bases(text)
    assert loads == 1 and short == []


def test_the_scan_sees_short_bases():
    written = "\tv_readfirstlane_b32 s5, v1\n"
    load = "\tglobal_load_lds_dwordx4 v0, s[4:5]\n"
    assert len(check_main_loops.short_bases(written + load)[1]) == 1
    assert len(check_main_loops.short_bases(written + "\ts_nop 0\n" + load)[1]) == 1
    assert len(check_main_loops.short_bases(written + "\ts_mov_b32 m0, s9\n\ts_nop 2\n" + load)[1]) == 1
    assert check_main_loops.short_bases(written + "\ts_nop 4\n" + load) == (1, [])
    assert check_main_loops.short_bases(written + "\ts_mov_b64 s[6:7], s[4:5]\n\tglobal_load_lds_dword v0, s[6:7]\n") == (1, [])
    assert check_main_loops.short_bases("\tv_mov_b32_e32 v4, v5\n\tglobal_load_lds_dwordx4 v[4:5], off\n") == (1, [])


def test_every_source_with_direct_loads_is_looked_at():
    """A file that issues them belongs to the script's list."""
    listed = {src for src, _ in check_main_loops.FILES}
    for name in os.listdir(build.CSRC):
        if name.endswith(".hip") and any(call in open(os.path.join(build.CSRC, name)).read() for call in ("dma16(", "dma4(", "global_load_lds")):
            assert name in listed, name
