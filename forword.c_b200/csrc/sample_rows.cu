// sample_rows.cu — C ABI of the sampling of rows: argument checks and launch.
#include <cuda_runtime.h>

#include "../../include/forword_b200.h"
#include "launch.h"
#include "sample_rows.cuh"

namespace fwb {
namespace {

template <typename T>
bool run_rows(SampleRowsArgs &k, uint32_t rows, cudaStream_t st) {
    // Blocks of a row: as many as a slice needs, and as keep the device's SMs
    // busy with the rows at hand while a slice is worth a block.
    const uint32_t sms = device_sms();
    uint32_t cluster = 1;
    while (cluster < kSrCluster && ((uint64_t)cluster * kSrSlice < k.n_vocab ||
                                    ((uint64_t)rows * cluster * 2 <= 2 * sms && cluster * 4096 < k.n_vocab)))
        cluster *= 2;
    k.slice = ((k.n_vocab + cluster - 1) / cluster + 7) / 8 * 8;
    k.vec = ((uintptr_t)k.logits | k.stride * sizeof(T)) % 16 == 0;
    static bool ready[64] = {};
    if (!opt_in(sample_rows_kernel<T>, sizeof(SrSmem), ready, "fwb_sample_rows")) return false;
    return launched(launch_after(sample_rows_kernel<T>, dim3(rows * cluster), kSrThreads, sizeof(SrSmem), cluster, st, k),
                    "fwb_sample_rows launch");
}

}  // namespace
}  // namespace fwb

using namespace fwb;

extern "C" int fwb_sample_rows_dev(const void *d_logits, uint32_t type, size_t n_row, size_t n_vocab, size_t row_stride,
                                   const float *d_uniform, const float *d_temperature, const int32_t *d_top_k,
                                   const float *d_top_p, const float *d_min_p, int32_t *d_token, float *d_logprob,
                                   void *stream) {
    if (!elem_bytes(type)) { fail("fwb_sample_rows: type must be 0 (F32), 1 (F16) or 30 (BF16)"); return -1; }
    if (!d_logits || !d_uniform || !d_token) { fail("fwb_sample_rows: null logits, uniform numbers or tokens"); return -1; }
    if (!n_row || !n_vocab) { fail("fwb_sample_rows: zero rows or tokens"); return -1; }
    if (n_vocab > kSrCluster * kSrSlice || n_row > 0x7fffffffu / kSrCluster) {
        fail("fwb_sample_rows: more than 262144 tokens, or too many rows");
        return -1;
    }
    if (row_stride < n_vocab && n_row > 1) { fail("fwb_sample_rows: row_stride smaller than n_vocab"); return -1; }
    if ((uintptr_t)d_logits % elem_bytes(type) ||
        ((uintptr_t)d_uniform | (uintptr_t)d_temperature | (uintptr_t)d_top_k | (uintptr_t)d_top_p | (uintptr_t)d_min_p |
         (uintptr_t)d_token | (uintptr_t)d_logprob) % 4) {
        fail("fwb_sample_rows: misaligned pointer");
        return -1;
    }
    SampleRowsArgs k{};
    k.logits = d_logits;
    k.stride = n_row > 1 ? row_stride : 0;
    k.n_vocab = (uint32_t)n_vocab;
    k.u = d_uniform; k.temp = d_temperature; k.top_k = d_top_k; k.top_p = d_top_p; k.min_p = d_min_p;
    k.token = d_token; k.logprob = d_logprob;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool ok = type == 0 ? run_rows<float>(k, (uint32_t)n_row, st)
                  : type == 1 ? run_rows<__half>(k, (uint32_t)n_row, st)
                              : run_rows<__nv_bfloat16>(k, (uint32_t)n_row, st);
    return ok ? 0 : -1;
}
