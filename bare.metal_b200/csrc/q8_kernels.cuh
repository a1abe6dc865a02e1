// Launchers of the 8-bit activation operators (q8_rows.cu, q8_matmul.cu). dtype 0 = fp32, 1 = bf16 (BMC_F32 / BMC_BF16).
// Arguments are checked by the entry points (backend_api.cu); every launcher enqueues on `st` and returns 0 or a negative code.
#pragma once
#include "common.cuh"

namespace bmb {

// widest row of the row kernels: one fp32 value per column in shared memory
constexpr int Q8_MAX_COLUMNS = 57344;

// Runs `setup` (0 = done, or a negative code) until it has succeeded once with the current device. The device is marked behind the set-up:
// of two threads whose first calls meet, none launches a kernel whose attributes the other is still setting (setting them twice is harmless).
template <typename Setup> int set_up_once(std::atomic<unsigned long long>& done_mask, const Setup& setup) {
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (done_mask.load(std::memory_order_acquire) & bit) return 0;
    const int rc = setup();
    if (rc == 0) done_mask.fetch_or(bit, std::memory_order_release);
    return rc;
}

int q8_quantize_rows(int dtype, int8_t* q, int ldq, float* scale, const void* x, int ldx, int rows, int C, cudaStream_t st);
// add, sum and their combination are optional (null); sum may be x or add
int q8_rmsnorm(int dtype, int8_t* q, int ldq, float* scale, void* sum, int lds, const void* x, int ldx, int add_dtype, const void* add, int lda,
               const float* w, int rows, int C, float eps, cudaStream_t st);
int q8_swiglu(int dtype, int8_t* q, int ldq, float* scale, const void* gate, const void* up, int ldgu, int rows, int H, cudaStream_t st);

// out[m, n] = (sum_k q[m, k] w[n, k]) * (scale[m] * wscale[n]) (+ residual[m, n])
int q8_matmul(int dtype, void* out, int ldo, const int8_t* q, int ldq, const float* scale, const int8_t* w, const float* wscale, const void* residual,
              int ldr, int M, int K, int N, int* err, cudaStream_t st);

}  // namespace bmb
