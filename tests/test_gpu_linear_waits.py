"""The dense products behind a kernel that lets them start early and runs longer than their bounded waits."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FRONT = r"""
#include <cuda_runtime.h>
// one warp: lets the next launch in the stream start, then sleeps until `ns` have passed (a million sleeps at most)
__global__ void front(long long ns) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (int i = 0; i < 1000000; ++i) {
    __nanosleep(10000);
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > ns) break;
  }
}
extern "C" int run_front(long long ns, void* stream) {
  front<<<1, 32, 0, (cudaStream_t)stream>>>(ns);
  return (int)cudaGetLastError();
}
"""


def test_a_long_launch_in_front(tmp_path):
    """Two and a half seconds in front, waits of one: no wait of the product runs out, the outputs are right."""
    from dsgx10_b200 import linear
    if shutil.which("nvcc") is None:
        pytest.skip("no nvcc on this machine")
    src, so = tmp_path / "front.cu", tmp_path / "front.so"
    src.write_text(FRONT)
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC", str(src), "-o", str(so)], check=True)
    lib = C.CDLL(os.fspath(so))
    lib.run_front.argtypes = [C.c_longlong, C.c_void_p]
    stream, status = torch.cuda.current_stream().cuda_stream, torch.zeros(1, dtype=torch.int32, device="cuda")
    for M, N, K in ((2, 40000, 1024), (16, 6144, 6144)):   # (longer than the rings: the weights must go on being asked for)
        b = torch.randint(0, 256, (-(-N // 8) * -(-K // 512), 2368), dtype=torch.uint8, device="cuda")
        b[:, 2048:2304].view(-1, 128, 2)[:, :, 1] = 0x3B
        w, x = linear.LinearW(N, K, b.view(-1)), torch.randn(M, K, device="cuda").bfloat16()
        want = linear.linear_decode(w, x)
        out = torch.zeros_like(want)
        torch.cuda.synchronize()
        assert lib.run_front(2_500_000_000, stream) == 0
        linear.linear_decode(w, x, out=out, status=status)
        torch.cuda.synchronize()
        assert int(status) == 0 and torch.equal(out, want)
