// Rows to 8 bits: code = rint(v / scale), scale = max|v| / 127 over the row, for v = x (bmc_quantize_rows_q8), v = RMSNorm(x + add) * w
// (bmc_rmsnorm_q8) and v = silu(gate) * up (bmc_swiglu_q8).
//
// The maximum is taken over the bit patterns of |v| as unsigned integers: they order like the values, and an infinity or NaN is larger than
// every number, so one reduction also says whether the row can be stored. A row that holds such a value gets the scale NaN (and codes 0),
// which every product with it carries on; a row whose scale would be subnormal (max|v| < 1.5e-36, a row of zeros among them) gets scale 0.
// No clamp is needed: scale and 1 / scale are each rounded once from normal numbers, so |v| / scale stays below 127 * (1 + 2^-22) and
// rounds to 127 at most.
//
// All three are bound by memory: every input is read once and every output written once, the row stays in registers between the reductions
// (up to 32 values a thread), so the threads of a row follow from its width. Against the measured copy rate: rows 32768 x 960 fp32 23.5 us
// (1.02), norm of an fp32 stream and a bf16 addend 52.9 us (1.00), SwiGLU 32768 x 2560 bf16 65.1 us (0.98); bf16 rows of middling widths 0.7
// to 0.85, where a row is too short for its block's phases. One block or warp per row, without a loop: blocks that stay and walk the rows
// were slower (62.8, 82 us), with a ring of bulk copies in front of them as well (56.5, 72 us).
#include "q8_kernels.cuh"

#include <cstdlib>
#include <type_traits>

namespace bmb {

namespace {

enum { Q8_ROWS = 0, Q8_NORM = 1, Q8_SWIGLU = 2 };

struct RowArgs {
    int8_t* q;
    float* scale;
    const void *x, *y;   // y: the addend (norm), the up projection (SwiGLU)
    void* sum;
    const float* w;
    int ldq, ldx, ldy, lds, C, rows;
    float eps;
};

constexpr uint32_t INF_BITS = 0x7f800000u;
__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// g / (1 + exp(-g)): the exponential is one special-function instruction on -g * log2(e) (relative error 2^-22 + 2 |g| 2^-24), the quotient
// a reciprocal and a product (2 units in the last place). For g < -88 the exponential is infinite and the quotient -0.
__device__ __forceinline__ float silu(float g) { return __fdividef(g, 1.0f + __expf(-g)); }

// scale and 1 / scale of a row whose largest |v| has the bit pattern `top`; inv = 0 where every code is 0
__device__ __forceinline__ float row_scale(uint32_t top, float& inv) {
    inv = 0.0f;
    if (top >= INF_BITS) return quiet_nan();
    const float s = __uint_as_float(top) / 127.0f;
    if (s < 1.17549435e-38f) return 0.0f;
    inv = 1.0f / s;
    return s;
}
// 1 / rms of a row. A sum of squares that overflowed has no reciprocal root: the row becomes NaN, not zero.
__device__ __forceinline__ float row_rstd(float ss, int C, float eps) {
    return ss < __uint_as_float(INF_BITS) ? 1.0f / sqrtf(ss / (float)C + eps) : quiet_nan();
}
// the code of v in the low byte: adding 1.5 * 2^23 leaves rint(v * inv) in the mantissa's low bits, in two's complement, without the
// conversion unit (a quarter of the rate). A NaN, which only a row with inv = 0 holds, is replaced before.
__device__ __forceinline__ uint32_t code_bits(float v, float inv) { return __float_as_uint(__fmaf_rn(v, inv, 12582912.0f)); }
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// N consecutive elements as floats, in the widest loads their size allows
template <typename T, int N> struct Pack;
template <typename T> struct Pack<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void unpack(float (&f)[1]) const { f[0] = to_f32(v); }
    __device__ __forceinline__ static void store(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};
template <> struct Pack<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *(const float4*)p; }
    __device__ __forceinline__ void unpack(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
    __device__ __forceinline__ static void store(float* p, const float (&f)[4]) { Vec<float>::store(p, f); }
};
template <> struct Pack<float, 8> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = *(const float4*)p; b = *(const float4*)(p + 4); }
    __device__ __forceinline__ void unpack(float (&f)[8]) const { f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w; }
};
template <> struct Pack<bf16, 4> {
    uint2 v;
    __device__ __forceinline__ void load(const bf16* p) { v = *(const uint2*)p; }
    __device__ __forceinline__ void unpack(float (&f)[4]) const {
        f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
        f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
    }
};
template <> struct Pack<bf16, 8> {
    uint4 v;
    __device__ __forceinline__ void load(const bf16* p) { v = Vec<bf16>::load_raw(p); }
    __device__ __forceinline__ void unpack(float (&f)[8]) const { Vec<bf16>::unpack(v, f); }
    __device__ __forceinline__ static void store(bf16* p, const float (&f)[8]) { Vec<bf16>::store(p, f); }
};

template <int N> __device__ __forceinline__ void store_codes(int8_t* p, const float (&f)[N], float inv) {
    if constexpr (N == 1) {
        *p = (int8_t)code_bits(f[0], inv);
    } else {
        uint32_t w[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = pack4(code_bits(f[4 * i], inv), code_bits(f[4 * i + 1], inv), code_bits(f[4 * i + 2], inv), code_bits(f[4 * i + 3], inv));
        if constexpr (N == 4) *(uint32_t*)p = w[0];
        else *(uint2*)p = make_uint2(w[0], w[1]);
    }
}

// Reductions over the threads of a row: one warp (WARP), or the block.
template <bool WARP> __device__ __forceinline__ float row_sum(float v, float* red) {
    v = warp_sum(v);
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = blockDim.x >> 5;
    return warp_sum((int)(threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0.0f);
}
template <bool WARP> __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = blockDim.x >> 5;
    return __reduce_max_sync(0xffffffffu, (int)(threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0u);
}

constexpr int WARP_ROWS = 4;   // rows per block where a warp has a row

// V gains from w[c ..], c = `off` (0 to 3) above a multiple of four: whole vectors, and a shift that is the same for every thread of a row.
// Nothing in the branch uses a loaded value, so that all of a thread's loads are in flight together.
template <int V> struct ShiftedGains {
    float t[V + 4];
    __device__ __forceinline__ void load(const float* w, int c, int off, int C) {
        const int b = c - off;
#pragma unroll
        for (int k = 0; k < V / 4; ++k) vector(w + b + 4 * k, 4 * k);
        if (b + V + 4 <= C) {
            vector(w + b + V, V);
        } else {
#pragma unroll
            for (int j = V; j < V + 3; ++j) t[j] = b + j < C ? w[b + j] : 0.0f;
        }
    }
    __device__ __forceinline__ void vector(const float* p, int at) {
        const float4 x = *(const float4*)p;
        t[at] = x.x; t[at + 1] = x.y; t[at + 2] = x.z; t[at + 3] = x.w;
    }
    __device__ __forceinline__ void get(float (&f)[V], int off) const {
        float u[V + 2];
#pragma unroll
        for (int j = 0; j < V + 2; ++j) u[j] = (off & 1) ? t[j + 1] : t[j];
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = (off & 2) ? u[j + 2] : u[j];
    }
};
// and where rows start on a vector
template <int V> struct Gains {
    Pack<float, V> v;
    __device__ __forceinline__ void load(const float* w, int c, int, int) { v.load(w + c); }
    __device__ __forceinline__ void get(float (&f)[V], int) const { v.unpack(f); }
};

// V elements per access, NV accesses per thread. WARP: a warp per row, WARP_ROWS rows per block; otherwise a block per row.
// EDGE: rows that do not start on a vector (an odd width), but on the same element of one in every operand: the vectors lie where memory has
// them, and the up to V - 1 elements in front of the first and behind the last are one element each of the first threads. (Their loads go out
// with the others. Vectors that hang over a row's ends, element by element in one lane, were slower: norm of 8192 x 4099
// bf16 + bf16 70.5 us against 52.7, rows 24.3 against 17.0.)
template <int MODE, typename TX, typename TY, int V, int NV, bool WARP, bool EDGE>
__global__ void __launch_bounds__(WARP ? 32 * WARP_ROWS : 512) q8_row_kernel(const RowArgs p) {
    __shared__ float red[32];
    __shared__ uint32_t redu[32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int row = WARP ? (int)blockIdx.x * WARP_ROWS + (int)(threadIdx.x >> 5) : (int)blockIdx.x;
    const int t = WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x, nt = WARP ? 32 : (int)blockDim.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= p.rows) return;   // whole warps only, and only where a warp has a row
    const TX* x = (const TX*)p.x + (size_t)row * p.ldx;
    const TY* y = (const TY*)p.y + (size_t)row * p.ldy;
    TX* sum = MODE == Q8_NORM && p.sum ? (TX*)p.sum + (size_t)row * p.lds : nullptr;
    int8_t* q = p.q + (size_t)row * p.ldq;
    const bool has_y = MODE == Q8_SWIGLU || (MODE == Q8_NORM && p.y != nullptr);
    const int front = EDGE ? (int)(-(uintptr_t)((uintptr_t)x / sizeof(TX)) & (V - 1)) : 0, back = EDGE ? (p.C - front) & (V - 1) : 0, end = p.C - back;
    const auto column = [&](int i) { return front + (t + i * nt) * V; };
    const bool single = EDGE && t < front + back;   // of 2 V - 2 at the most: a row has 32 threads or more
    const int cs = t < front ? t : end + t - front;
    const auto value = [&](float a, float b) { return !has_y ? a : MODE == Q8_SWIGLU ? silu(a) * b : a + b; };
    Pack<TX, V> px[NV];
    Pack<TY, V> py[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = column(i);
        if (c < end) {
            px[i].load(x + c);
            if (has_y) py[i].load(y + c);
        }
    }
    float v[NV][V], one = 0.0f;
    if (single) one = value(to_f32(x[cs]), has_y ? to_f32(y[cs]) : 0.0f);
    float ss = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = column(i);
        if (c < end) {
            px[i].unpack(v[i]);
            if (has_y) {
                float f[V];
                py[i].unpack(f);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] = value(v[i][j], f[j]);
            }
            if (sum) Pack<TX, V>::store(sum + c, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (MODE == Q8_NORM) ss = fmaf(v[i][j], v[i][j], ss);
            else top = max(top, abs_bits(v[i][j]));
        }
    }
    if (EDGE) {
        if (single && sum) sum[cs] = from_f32<TX>(one);
        if (MODE == Q8_NORM) ss = fmaf(one, one, ss);
        else top = max(top, abs_bits(one));
    }
    if (MODE == Q8_NORM) {
        std::conditional_t<EDGE, ShiftedGains<V>, Gains<V>> w[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (column(i) < end) w[i].load(p.w, column(i), front & 3, p.C);
        const float w1 = single ? p.w[cs] : 0.0f;
        const float r = row_rstd(row_sum<WARP>(ss, red), p.C, p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (column(i) < end) {
                float g[V];
                w[i].get(g, front & 3);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[i][j] = v[i][j] * r * g[j];
                    top = max(top, abs_bits(v[i][j]));
                }
            }
        }
        if (single) {
            one = one * r * w1;
            top = max(top, abs_bits(one));
        }
    }
    float inv;
    const float s = row_scale(row_max<WARP>(top, redu), inv);
    if (t == 0) p.scale[row] = s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = column(i);
        if (c < end) {
            if (inv == 0.0f)
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] = 0.0f;
            store_codes<V>(q + c, v[i], inv);
        }
    }
    if (single) q[cs] = inv == 0.0f ? 0 : (int8_t)code_bits(one, inv);
}

// Rows that 512 threads cannot hold in registers: a block per row, the row in shared memory between the passes.
template <int MODE, typename TX, typename TY>
__global__ void __launch_bounds__(1024) q8_wide_row_kernel(const RowArgs p) {
    extern __shared__ float v[];
    __shared__ float red[32];
    __shared__ uint32_t redu[32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
            ss = fmaf(f, f, ss);
        }
        v[c] = f;
        top = max(top, abs_bits(f));
    }
    if (MODE == Q8_NORM) {
        const float r = row_rstd(row_sum<false>(ss, red), p.C, p.eps);
        top = 0;
        for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
            const float f = v[c] * r * p.w[c];
            v[c] = f;
            top = max(top, abs_bits(f));
        }
    }
    float inv;
    const float s = row_scale(row_max<false>(top, redu), inv);
    if (threadIdx.x == 0) p.scale[row] = s;
    int8_t* q = p.q + row * p.ldq;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) q[c] = inv == 0.0f ? 0 : (int8_t)code_bits(v[c], inv);
}

// Every kernel here waits for its predecessor itself (griddepcontrol.wait), so it may be launched while that one still runs.
template <typename K> int launch(K kernel, unsigned grid, unsigned block, size_t smem, const RowArgs& p, cudaStream_t st) {
    static const bool overlap = getenv("BM_NO_PDL") == nullptr;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = overlap ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess) return 0;
    cudaGetLastError();   // a launch that failed must not poison the status of later calls
    return -9;
}

template <int MODE, typename TX, typename TY, int V, int NV, bool EDGE> int launch_rows(const RowArgs& p, int threads, cudaStream_t st) {
    if (threads == 32)
        return launch(q8_row_kernel<MODE, TX, TY, V, NV, true, EDGE>, ((unsigned)p.rows + WARP_ROWS - 1) / WARP_ROWS, 32 * WARP_ROWS, 0, p, st);
    return launch(q8_row_kernel<MODE, TX, TY, V, NV, false, EDGE>, (unsigned)p.rows, (unsigned)threads, 0, p, st);
}

// Threads per row. Many rows: 32 or 16 values a thread, whichever leaves fewer of the row's threads idle (loads in flight are what counts:
// 32768 x 960 fp32 with a warp per row 23.5 us, with 16 or 8 values a thread 34); SwiGLU, which loads two vectors for each value, two accesses
// (32768 x 2560 bf16 60 to 65 us, four accesses 64 to 68, one 79); bf16 rows of 1024 to 2048 columns 64 values, a warp per row (16384 x 1536
// 13.7 us against 17.7). Few rows: as many threads as there are vectors, so that a row costs one load's latency and two reductions.
template <int MODE, typename TX, typename TY, int V, bool EDGE> int launch_vec(const RowArgs& p, cudaStream_t st) {
    const int vecs = EDGE ? p.C / V : (p.C + V - 1) / V;
    constexpr bool LONG = MODE == Q8_ROWS && V == 8 && !EDGE;
    constexpr int MOST = V == 1 ? 16 : LONG ? 8 : 32 / V;   // accesses per thread (single elements: 16, or a block could not have 512 threads)
    const auto threads_for = [&](int n) { return ((vecs + n - 1) / n + 31) / 32 * 32; };
    const bool one_warp = LONG && vecs > 128 && vecs <= 256;
    int nv = LONG && !one_warp ? MOST / 2 : MOST;
    if (MODE == Q8_SWIGLU && V > 1) nv = 2;
    if (MODE == Q8_NORM && EDGE) nv = MOST / 2;   // shifted gains hold up to twice the registers: 8192 x 4099 fp32 + bf16 61.9 us against 68.6
    while (threads_for(nv) > 512) nv *= 2;
    if (!one_warp && threads_for(nv / 2) <= 512 && threads_for(nv / 2) * (nv / 2) < threads_for(nv) * nv) nv /= 2;
    while (nv > 1 && threads_for(nv / 2) <= 512 && (long)p.rows * threads_for(nv) < 148L * 512) nv /= 2;
    const int threads = threads_for(nv);
    if constexpr (MOST >= 16) {
        if (nv > 8) return launch_rows<MODE, TX, TY, V, 16, EDGE>(p, threads, st);
    }
    if constexpr (MOST >= 8) {
        if (nv > 4) return launch_rows<MODE, TX, TY, V, 8, EDGE>(p, threads, st);
    }
    if (nv > 2) return launch_rows<MODE, TX, TY, V, 4, EDGE>(p, threads, st);
    if (nv > 1) return launch_rows<MODE, TX, TY, V, 2, EDGE>(p, threads, st);
    return launch_rows<MODE, TX, TY, V, 1, EDGE>(p, threads, st);
}

template <int MODE, typename TX, typename TY> int run_rows(const RowArgs& p, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(TX);
    constexpr int SCALAR_MOST = 16 * 512, VEC_MOST = 32 * 512;
    const auto wide = [&]() {
        static std::atomic<unsigned long long> done{0};
        const int rc = set_up_once(done, [] {
            return cudaFuncSetAttribute(q8_wide_row_kernel<MODE, TX, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q8_MAX_COLUMNS * 4) == cudaSuccess ? 0 : -5;
        });
        if (rc) return rc;
        return launch(q8_wide_row_kernel<MODE, TX, TY>, (unsigned)p.rows, 1024, (size_t)p.C * 4, p, st);
    };
    // Vectors of 16 bytes of x, and as many elements of everything else, where every row of every operand starts on such a boundary, or on the
    // same element behind one (contiguous tensors of an odd width). Others go element by element.
    const auto begins = [](const void* ptr, size_t elem) { return (int)((uintptr_t)ptr / elem % V); };
    const int at = begins(p.x, sizeof(TX)), step = p.ldx % V;
    const bool same = begins(p.q, 1) == at && p.ldq % V == step && (!p.y || (begins(p.y, sizeof(TY)) == at && p.ldy % V == step)) &&
                      (!p.sum || (begins(p.sum, sizeof(TX)) == at && p.lds % V == step)) && (!p.w || (uintptr_t)p.w % 16 == 0);
    const bool vec = same && at == 0 && step == 0 && p.C % V == 0;
    if (p.C / V > VEC_MOST / V || (!same && p.C > SCALAR_MOST)) return wide();
    if (vec) return launch_vec<MODE, TX, TY, V, false>(p, st);
    return same && p.C >= 8 * V ? launch_vec<MODE, TX, TY, V, true>(p, st) : launch_vec<MODE, TX, TY, 1, false>(p, st);
}

}  // namespace

int q8_quantize_rows(int dtype, int8_t* q, int ldq, float* scale, const void* x, int ldx, int rows, int C, cudaStream_t st) {
    RowArgs p{q, scale, x, nullptr, nullptr, nullptr, ldq, ldx, 0, 0, C, rows, 0.0f};
    return dtype ? run_rows<Q8_ROWS, bf16, bf16>(p, st) : run_rows<Q8_ROWS, float, float>(p, st);
}

int q8_rmsnorm(int dtype, int8_t* q, int ldq, float* scale, void* sum, int lds, const void* x, int ldx, int add_dtype, const void* add, int lda,
               const float* w, int rows, int C, float eps, cudaStream_t st) {
    RowArgs p{q, scale, x, add, sum, w, ldq, ldx, lda, lds, C, rows, eps};
    if (dtype) return add_dtype ? run_rows<Q8_NORM, bf16, bf16>(p, st) : run_rows<Q8_NORM, bf16, float>(p, st);
    return add_dtype ? run_rows<Q8_NORM, float, bf16>(p, st) : run_rows<Q8_NORM, float, float>(p, st);
}

int q8_swiglu(int dtype, int8_t* q, int ldq, float* scale, const void* gate, const void* up, int ldgu, int rows, int H, cudaStream_t st) {
    RowArgs p{q, scale, gate, up, nullptr, nullptr, ldq, ldgu, ldgu, 0, H, rows, 0.0f};
    return dtype ? run_rows<Q8_SWIGLU, bf16, bf16>(p, st) : run_rows<Q8_SWIGLU, float, float>(p, st);
}

}  // namespace bmb
