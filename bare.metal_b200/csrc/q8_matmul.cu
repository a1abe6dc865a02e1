// Product of 8-bit integer matrices with a scale per row of each (per token and per output channel):
//   out[m, n] = (sum_k q[m, k] w[n, k]) * (scale[m] * wscale[n]) (+ residual[m, n])
// The sum is an exact 32-bit integer for every K up to 131071 (|q w| <= 2^14), so the only roundings are the conversion of the sum, the
// product of the scales, their product, the residual's addition and the store: the result does not depend on the order of the sum.
#include "q8_kernels.cuh"

namespace bmb {

namespace {

constexpr int T = 64, KT = 64;   // tile of the output, and of K per step

template <typename TO>
__global__ void __launch_bounds__(256) q8_matmul_kernel(TO* out, int ldo, const int8_t* q, int ldq, const float* scale, const int8_t* w,
                                                        const float* wscale, const TO* residual, int ldr, int M, int K, int N, int tiles_n) {
    __shared__ int sq[T][KT / 4 + 1], sw[T][KT / 4 + 1];
    const int m0 = (int)(blockIdx.x / tiles_n) * T, n0 = (int)(blockIdx.x % tiles_n) * T;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += KT) {
        const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
        const int4 z = make_int4(0, 0, 0, 0);
        const int4 a = m0 + r < M && k0 + c < K ? *(const int4*)(q + (size_t)(m0 + r) * ldq + k0 + c) : z;
        const int4 b = n0 + r < N && k0 + c < K ? *(const int4*)(w + (size_t)(n0 + r) * K + k0 + c) : z;
        int* da = &sq[r][c / 4];
        int* db = &sw[r][c / 4];
        da[0] = a.x; da[1] = a.y; da[2] = a.z; da[3] = a.w;
        db[0] = b.x; db[1] = b.y; db[2] = b.z; db[3] = b.w;
        __syncthreads();
        for (int k = 0; k < KT / 4; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sq[ty + 16 * i][k], sw[tx + 16 * j][k], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m < M && n < N) {
                float f = (float)acc[i][j] * (scale[m] * wscale[n]);
                if (residual) f += to_f32(residual[(size_t)m * ldr + n]);
                out[(size_t)m * ldo + n] = from_f32<TO>(f);
            }
        }
}

}  // namespace

int q8_matmul(int dtype, void* out, int ldo, const int8_t* q, int ldq, const float* scale, const int8_t* w, const float* wscale, const void* residual,
              int ldr, int M, int K, int N, int* err, cudaStream_t st) {
    (void)err;
    const int tiles_n = (N + T - 1) / T;
    const long tiles = (long)((M + T - 1) / T) * tiles_n;
    if (tiles > 0x7fffffffL) return -1;
    if (dtype) q8_matmul_kernel<bf16><<<(unsigned)tiles, 256, 0, st>>>((bf16*)out, ldo, q, ldq, scale, w, wscale, (const bf16*)residual, ldr, M, K, N, tiles_n);
    else q8_matmul_kernel<float><<<(unsigned)tiles, 256, 0, st>>>((float*)out, ldo, q, ldq, scale, w, wscale, (const float*)residual, ldr, M, K, N, tiles_n);
    return cudaGetLastError() == cudaSuccess ? 0 : -9;
}

}  // namespace bmb
