"""GPU: the bounded waits of the beam-search kernels when they run out.  A small
kernel built from the library's own headers waits for a barrier that completes
late or not at all; the error word is set beforehand, so that a wait gives up
after its first thousand polls.  And the error word itself (beam_status.cuh)."""
import ctypes
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forword.c_b200", "csrc")

SOURCE = r"""
#include "beam_status.cuh"
#include "common.cuh"
using namespace fwb;

// Warp 0 waits; warp 1 arrives after `delay` cycles, or not at all.
__global__ void wait_kernel(uint32_t *err, long long delay, uint32_t *answers) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        fence_mbar_init();
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        answers[threadIdx.x] = mbar_wait_warp(&bar, 0, err, ERR_WAIT_FULL) ? 1u : 0u;
    } else if (threadIdx.x == 32 && delay >= 0) {
        const long long t = clock64();
        for (int i = 0; i < 1 << 22 && clock64() - t < delay; ++i) {}
        mbar_arrive(&bar);
    }
    __syncthreads();
}

extern "C" int wait_run(unsigned preset, long long delay, uint32_t *answers, uint32_t *err) {
    uint32_t *d = nullptr;
    if (cudaMalloc(&d, 33 * 4) != cudaSuccess) return -1;
    cudaMemset(d, 0xff, 32 * 4);
    cudaMemcpy(d + 32, &preset, 4, cudaMemcpyHostToDevice);
    wait_kernel<<<1, 64>>>(d + 32, delay, d);
    cudaMemcpy(answers, d, 32 * 4, cudaMemcpyDeviceToHost);
    const cudaError_t e = cudaMemcpy(err, d + 32, 4, cudaMemcpyDeviceToHost);
    cudaFree(d);
    return (int)e;
}

__global__ void set_kernel(uint32_t bit) { atomicOr(&g_beam_err, 1u << bit); }

// Errors set one after the other on one stream while another looks: all that was seen.
extern "C" int status_run(int rounds, uint32_t *seen, uint32_t *left) {
    cudaStream_t a, b;
    if (cudaStreamCreateWithFlags(&a, cudaStreamNonBlocking) != cudaSuccess ||
        cudaStreamCreateWithFlags(&b, cudaStreamNonBlocking) != cudaSuccess)
        return -1;
    int bad = 0;
    for (int r = 0; r < rounds; ++r) {
        uint32_t all = 0, word = 0;
        for (uint32_t bit = 0; bit < 32; ++bit) {
            set_kernel<<<1, 1, 0, b>>>(bit);
            if (beam_take_status(a, word) != cudaSuccess) return -1;
            all |= word;
        }
        if (cudaStreamSynchronize(b) != cudaSuccess || beam_take_status(a, word) != cudaSuccess) return -1;
        all |= word;
        bad += all != 0xffffffffu;
        *seen = all;
        if (beam_take_status(b, *left) != cudaSuccess) return -1;
        bad += *left != 0;
    }
    cudaStreamDestroy(a);
    cudaStreamDestroy(b);
    return bad;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("waits")
    (d / "waits.cu").write_text(SOURCE)
    so = d / "libwaits.so"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "-shared", "-cudart", "static",
                    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-I", CSRC, "-o", str(so), str(d / "waits.cu")],
                   check=True, capture_output=True)
    return ctypes.CDLL(str(so))


def run(lib, preset, delay):
    answers, err = (ctypes.c_uint32 * 32)(), ctypes.c_uint32()
    assert lib.wait_run(ctypes.c_uint32(preset), ctypes.c_longlong(delay), answers, ctypes.byref(err)) == 0
    return set(answers), err.value


def test_a_wait_that_is_met(lib):
    for delay in (0, 1000, 20000):
        assert run(lib, 0, delay) == ({1}, 0)


def test_a_wait_that_runs_out(lib):
    """Every lane gives up; another's error stays as it is."""
    for word in (1, 1 << 6):
        assert run(lib, word, -1) == ({0}, word)


def test_lanes_answer_alike(lib):
    """The barrier completes about when the lanes give up, sooner and later: one answer for the warp."""
    seen = set()
    for delay in list(range(0, 400000, 1500)) + list(range(400000, 4000000, 40000)):
        answers, _ = run(lib, 1, delay)
        assert len(answers) == 1 and answers <= {0, 1}
        seen |= answers
    assert 1 in seen


def test_no_error_is_lost_between_streams(lib):
    """Each look takes what was set until then, and leaves what is set later to the next."""
    seen, left = ctypes.c_uint32(), ctypes.c_uint32(1)
    assert lib.status_run(200, ctypes.byref(seen), ctypes.byref(left)) == 0
    assert seen.value == 0xffffffff and left.value == 0
