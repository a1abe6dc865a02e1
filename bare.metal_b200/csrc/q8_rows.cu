// Rows to 8 bits: code = rint(v / scale), scale = max|v| / 127 over the row, for v = x (bmc_quantize_rows_q8), v = RMSNorm(x + add) * w
// (bmc_rmsnorm_q8) and v = silu(gate) * up (bmc_swiglu_q8).
//
// The maximum is taken over the bit patterns of |v| as unsigned integers: they order like the values, and an infinity or NaN is larger than
// every number, so one reduction also says whether the row can be stored. A row that holds such a value gets the scale NaN (and codes 0),
// which every product with it carries on; a row whose scale would be subnormal (max|v| < 1.5e-36, a row of zeros among them) gets scale 0.
// No clamp is needed: scale, 1 / scale and the product are each rounded once from normal numbers, so |v| / scale stays below
// 127 * (1 + 2^-22) and rounds to 127 at most.
#include "q8_kernels.cuh"

namespace bmb {

namespace {

enum { Q8_ROWS = 0, Q8_NORM = 1, Q8_SWIGLU = 2 };

struct RowArgs {
    int8_t* q;
    float* scale;
    const void *x, *y;   // y: the addend (norm), the up projection (SwiGLU)
    void* sum;
    const float* w;
    int ldq, ldx, ldy, lds, C;
    float eps;
};

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
    __syncthreads();
    return t;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    uint32_t t = 0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t = max(t, red[i]);
    return t;
}

// scale and 1 / scale of a row whose largest |v| has the bit pattern `top`
__device__ __forceinline__ float row_scale(uint32_t top, float& inv) {
    if (top >= 0x7f800000u) {
        inv = 0.0f;
        return __uint_as_float(0x7fc00000u);
    }
    const float s = __uint_as_float(top) / 127.0f;
    if (s < 1.17549435e-38f) {
        inv = 0.0f;
        return 0.0f;
    }
    inv = 1.0f / s;
    return s;
}

// One block per row, the row's values in shared memory between the passes.
template <int MODE, typename TX, typename TY>
__global__ void __launch_bounds__(256) q8_row_kernel(const RowArgs p) {
    extern __shared__ float v[];
    __shared__ float red[8];
    __shared__ uint32_t redu[8];
    const size_t row = blockIdx.x;
    const TX* x = (const TX*)p.x + row * p.ldx;
    const TY* y = p.y ? (const TY*)p.y + row * p.ldy : nullptr;
    float ss = 0.0f;
    uint32_t top = 0;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
        float f = to_f32(x[c]);
        if (MODE == Q8_SWIGLU) f = silu(f) * to_f32(y[c]);
        if (MODE == Q8_NORM) {
            if (y) f += to_f32(y[c]);
            if (p.sum) ((TX*)p.sum)[row * p.lds + c] = from_f32<TX>(f);
            ss += f * f;
        }
        v[c] = f;
        top = max(top, __float_as_uint(f) & 0x7fffffffu);
    }
    if (MODE == Q8_NORM) {
        ss = block_sum(ss, red);
        // a sum of squares that overflowed has no reciprocal root: the row becomes NaN, not zero
        const float r = ss < __uint_as_float(0x7f800000u) ? 1.0f / sqrtf(ss / (float)p.C + p.eps) : __uint_as_float(0x7fc00000u);
        top = 0;
        for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
            const float f = v[c] * r * p.w[c];
            v[c] = f;
            top = max(top, __float_as_uint(f) & 0x7fffffffu);
        }
    }
    top = block_max(top, redu);
    float inv;
    const float s = row_scale(top, inv);
    if (threadIdx.x == 0) p.scale[row] = s;
    int8_t* q = p.q + row * p.ldq;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) q[c] = inv == 0.0f ? 0 : (int8_t)__float2int_rn(v[c] * inv);
}

template <int MODE, typename TX, typename TY>
int launch(const RowArgs& p, int rows, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    if (first_use_on_current_device(done))
        if (cudaFuncSetAttribute(q8_row_kernel<MODE, TX, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q8_MAX_COLUMNS * 4) != cudaSuccess) return -5;
    q8_row_kernel<MODE, TX, TY><<<rows, 256, (size_t)p.C * 4, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? 0 : -9;
}

}  // namespace

int q8_quantize_rows(int dtype, int8_t* q, int ldq, float* scale, const void* x, int ldx, int rows, int C, cudaStream_t st) {
    RowArgs p{q, scale, x, nullptr, nullptr, nullptr, ldq, ldx, 0, 0, C, 0.0f};
    return dtype ? launch<Q8_ROWS, bf16, bf16>(p, rows, st) : launch<Q8_ROWS, float, float>(p, rows, st);
}

int q8_rmsnorm(int dtype, int8_t* q, int ldq, float* scale, void* sum, int lds, const void* x, int ldx, int add_dtype, const void* add, int lda,
               const float* w, int rows, int C, float eps, cudaStream_t st) {
    RowArgs p{q, scale, x, add, sum, w, ldq, ldx, lda, lds, C, eps};
    if (dtype) return add_dtype ? launch<Q8_NORM, bf16, bf16>(p, rows, st) : launch<Q8_NORM, bf16, float>(p, rows, st);
    return add_dtype ? launch<Q8_NORM, float, bf16>(p, rows, st) : launch<Q8_NORM, float, float>(p, rows, st);
}

int q8_swiglu(int dtype, int8_t* q, int ldq, float* scale, const void* gate, const void* up, int ldgu, int rows, int H, cudaStream_t st) {
    RowArgs p{q, scale, gate, up, nullptr, nullptr, ldq, ldgu, ldgu, 0, H, 0.0f};
    return dtype ? launch<Q8_SWIGLU, bf16, bf16>(p, rows, st) : launch<Q8_SWIGLU, float, float>(p, rows, st);
}

}  // namespace bmb
