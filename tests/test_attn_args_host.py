"""The addresses that the host makes for the attention over quantised pages, compiled for the host only."""
import subprocess

from test_capi import ROOT

SOURCE = """
#include <hip/hip_runtime.h>
#include <cstdio>
namespace nova { namespace { constexpr int kMinPiece = 3, kGroupTiles = 4; } }
#include "attn_ragged.h"
int main() {
    const int layer = nova::Model::L - 1, nb = 1 << 27, page = 2176;
    alignas(16) static unsigned char some[16];
    const auto* f = reinterpret_cast<const float*>(some);
    auto* base = reinterpret_cast<uint8_t*>((uintptr_t)1 << 40);
    const nova::AttnArgs a = nova::attn_args(page, f, base, (const int32_t*)some, 4, (const int32_t*)some, 2, layer, nb, (float*)some);
    std::printf("%lld %lld\\n", (long long)(a.pool - base), (long long)layer * nb * page);
}
"""


def test_a_layers_first_page_past_32_bits_of_pages(tmp_path):
    """layers times pages beyond 2^31"""
    src, exe = tmp_path / "args.hip", tmp_path / "args"
    src.write_text(SOURCE)
    kernels = ROOT / "conflux-nova_amd" / "code" / "kernel" / "hip"
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-host-only", "-std=c++17", "-O1", "-DNOVA_MODEL_QWEN25_7B", f"-I{ROOT / 'include'}",
                    f"-I{kernels.parent.parent}", f"-I{kernels}", str(src), "-o", str(exe)], check=True, capture_output=True)
    got, want = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert got == want
