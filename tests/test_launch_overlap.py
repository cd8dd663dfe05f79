"""B200_GEMM_NO_PDL: every kernel of the library starts only after the one before it in the stream."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent
CSRC = REPO / "h100_gemm_b200" / "csrc"

CHAIN = """
import ctypes
import torch
import h100_gemm_b200 as g

x = torch.randn(4, 256, device="cuda").bfloat16()
w1, w2 = torch.randn(2, 128, 256, device="cuda").bfloat16(), torch.randn(2, 256, 64, device="cuda").bfloat16()
router = torch.randn(2, 256, device="cuda").bfloat16()
q, w = g.quantize_mx(x), g.quantize_mx(torch.randn(256, 256, device="cuda").bfloat16())
y, z, v, u = (torch.empty(4, 256, dtype=torch.bfloat16, device="cuda") for _ in range(4))
work = torch.empty(g.moe_workspace_bytes(4, 2, 1, 256, 64), dtype=torch.uint8, device="cuda")
b = torch.randn(256, 256, device="cuda").bfloat16()

def chain(s):
    g.quantize_mx(x, out=q, stream=s)
    g.gemm_mx(q, w, out=y, stream=s)
    g.moe_layer(y, router, w1, w2, 1, out=z, workspace=work, stream=s)
    g.dequantize_mx(q, out=v, stream=s)
    g.gemm(v, b, out=u, stream=s)

stream = torch.cuda.Stream()
chain(stream)
torch.cuda.synchronize()

rt = ctypes.CDLL("libcudart.so.12")
handle, graph, count = ctypes.c_void_p(stream.cuda_stream), ctypes.c_void_p(), ctypes.c_size_t()
assert rt.cudaStreamBeginCapture(handle, 2) == 0  # relaxed
chain(stream)
assert rt.cudaStreamEndCapture(handle, ctypes.byref(graph)) == 0
assert rt.cudaGraphGetEdges_v2(graph, None, None, None, ctypes.byref(count)) == 0
ends = [(ctypes.c_void_p * count.value)() for _ in range(2)]
data = (ctypes.c_ubyte * (8 * count.value))()     # from_port, to_port, type, 5 reserved bytes
assert rt.cudaGraphGetEdges_v2(graph, *ends, data, ctypes.byref(count)) == 0
print("edges", count.value, "programmatic", sum(t == 1 for t in data[2::8]))
"""


def test_one_place_decides_on_overlap():
    """No launch sets the attribute by itself."""
    found = [(path.name, line.strip()) for path in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.h")])
             for line in path.read_text().splitlines() if "programmaticStreamSerializationAllowed" in line]
    assert found and all(line.endswith("programmatic_launch();") for _, line in found), found


@pytest.mark.gpu
@pytest.mark.parametrize("off", [False, True])
def test_switch_reaches_every_kernel(off):
    """A captured chain of all operators: seven kernels, six edges between them, programmatic or none of them."""
    env = {k: v for k, v in os.environ.items() if k != "B200_GEMM_NO_PDL"}
    if off:
        env["B200_GEMM_NO_PDL"] = "1"
    done = subprocess.run([sys.executable, "-c", CHAIN], cwd=REPO, env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert done.stdout.split()[-4:] == ["edges", "6", "programmatic", "0" if off else "6"], done.stdout
