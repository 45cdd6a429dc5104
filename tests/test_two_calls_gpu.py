"""Calls of the C entry points from host threads at once, without Python's lock between them."""
import ctypes
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu

SOURCE = r"""
#include <atomic>
#include <cstdint>
#include <thread>
using Route = int (*)(const void*, int, int64_t, const float*, const uint8_t*, float*, int32_t*, int32_t*, int64_t, int64_t,
                      int64_t, int, int64_t, int64_t, int, double, void*);
// Two threads, n calls each with experts, inputs, outputs and a stream of its own; refused[t]: its calls that failed.
extern "C" void two(void* route, const void** x, const float** b, float** w, int32_t** e, const int64_t* E, void** stream,
                    int64_t N, int64_t k, int n, int* refused) {
  std::atomic<int> here{0};
  const auto work = [&](int t) {
    ++here;
    while (here < 2) {}
    for (int i = 0; i < n; ++i)
      refused[t] += reinterpret_cast<Route>(route)(x[t], 0, E[t], b[t], nullptr, w[t], e[t], nullptr, N, E[t], k, 0, 1, 1, 1,
                                                   1.0, stream[t]) != 0;
  };
  std::thread one(work, 0), two(work, 1);
  one.join();
  two.join();
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
@pytest.mark.parametrize("counts", [(260, 512), (520, 1024)])
def test_route_of_two_numbers_of_experts_at_once(tmp_path, counts):
    """Calls that run the same kernel with workspaces of other sizes: none is refused, each has its own results."""
    import streamtopk_sae as stk
    from streamtopk_sae import _capi
    (tmp_path / "two.cpp").write_text(SOURCE)
    so = tmp_path / "two.so"
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-pthread", "-o", so, tmp_path / "two.cpp"], check=True)
    N, k, n = 8, 4, 40000
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn(N, E, generator=gen, device="cuda") for E in counts]
    b = [torch.randn(E, generator=gen, device="cuda") * 0.1 for E in counts]
    w = [torch.zeros(N, k, device="cuda") for _ in counts]
    e = [torch.zeros(N, k, dtype=torch.int32, device="cuda") for _ in counts]
    streams = [torch.cuda.Stream() for _ in counts]
    torch.cuda.synchronize()

    def pointers(of):
        return (ctypes.c_void_p * 2)(*of)

    refused = (ctypes.c_int * 2)()
    lib = ctypes.CDLL(str(so))
    lib.two(ctypes.cast(_capi.load().stk_route_forward, ctypes.c_void_p), *(pointers([t.data_ptr() for t in ts])
            for ts in (x, b, w, e)), (ctypes.c_int64 * 2)(*counts), pointers([s.cuda_stream for s in streams]),
            ctypes.c_int64(N), ctypes.c_int64(k), n, refused)
    torch.cuda.synchronize()
    assert list(refused) == [0, 0]
    for i in range(2):
        ww, ee = stk.route_experts(x[i], k, bias=b[i])
        assert torch.equal(w[i], ww) and torch.equal(e[i], ee)
