// Product of 8-bit integer matrices with a scale per row of each (per token and per output channel):
//   out[m, n] = (sum_k q[m, k] w[n, k]) * (scale[m] * wscale[n]) (+ residual[m, n])
// The sum is an exact 32-bit integer for every K up to 131056 (|q w| <= 2^14), so the only roundings are the conversion of the sum, the
// product of the scales, their product, the residual's addition and the store: the result does not depend on the order of the sum, and a
// reduction split over several CTAs is as exact (and as reproducible) as one that is not.
//
// The tensor-core kernels compute the transposed tile: the weights are the A operand (128 output channels = the 128 lanes of tensor memory),
// the tokens the B operand (16 to 256 of them = accumulator columns). A warp then holds 32 consecutive channels of one token in one register
// across its lanes, so that a plain store of that register is a contiguous 128-byte (fp32) or 64-byte (bf16) piece of an output row whatever
// its alignment, the channel's scale is a register of the lane and the token's a broadcast from shared memory. Few tokens cost a narrow
// instruction instead of an empty tile.
//   q8_few_kernel    one to four tokens, without tensor cores: a warp per channel. 1 x 960 -> 1600 1.55 us.
//   q8_split_kernel  one tile of 128 channels per cluster; the CTAs of the cluster split K and exchange their partial sums through
//                    distributed shared memory. For outputs of too few tiles to fill the GPU: decode, short prompts. 64 x 2560 -> 960 with a
//                    residual 4.2 us: 0.8 until the first bytes are there, 1.2 for five k-blocks, 0.6 for the exchange, 0.3 for the stores.
//   q8_pair_kernel   persistent CTA pairs with tiles of 256 channels x up to 256 tokens, for everything larger. 8192 x 8192 -> 8192 341 us
//                    (3.22 POP/s, 0.97 of twice the measured bf16 rate), 32768 x 960 -> 5120 131 to 137 us.
#include "q8_kernels.cuh"

#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "ptx_sm100.cuh"

namespace bmb {

namespace {

constexpr int BM = 128;                   // channels per CTA
constexpr int BK = 128;                   // codes per k-block: one 128-byte swizzled row
constexpr int UK = 32;                    // codes per instruction
constexpr int A_BYTES = BM * BK;          // 16 KB
constexpr int NUM_THREADS = 192;          // split kernel: warp 0 copies, warp 1 issues the products, warps 2 to 5 are the epilogue (lane quarter = warp & 3)
constexpr int MAX_STAGES = 8;

struct Q8Args {
    void* out;
    const void* residual;
    const float *scale, *wscale;
    int ldo, ldr, M, N, K;     // M tokens, N channels
    int bn;                    // tokens per tile
    int tiles_ch, tiles_tok, kb_total;
    int splits, kb_per, stages;   // split kernel
    int* err;
};

__device__ __forceinline__ void store_pair(float* a, float* b, float2 v) {
    *a = v.x;
    *b = v.y;
}
__device__ __forceinline__ void store_pair(bf16* a, bf16* b, float2 v) {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    *a = h.x;
    *b = h.y;
}

// The residual of one channel and up to 32 consecutive tokens, as stored (widened where it is added: a conversion here would wait for the
// load). Always read before the first of these tokens is stored: out may be the residual.
template <typename TO> __device__ __forceinline__ void load_residual(const Q8Args& p, int m, int n, TO (&f)[32], int tokens) {
    const TO* res = (const TO*)p.residual + (size_t)m * p.ldr + n;
    const size_t step = p.ldr;
    if (tokens >= 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i, res += step) f[i] = *res;
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i, res += step)
            if (i < tokens) f[i] = *res;
    }
}
// One channel (this lane's) of up to 32 consecutive tokens: accumulators r, residual f, token scales sa. The epilogue's instructions are what a
// short reduction waits for (with K = 960 a tile's products take 3840 cycles): whole chunks run without bounds (with a bound per token the
// compiler made 21 instructions of each), two tokens per multiplication and conversion.
template <typename TO, bool RES>
__device__ __forceinline__ void store_tokens(const Q8Args& p, int m, int n, const uint32_t (&r)[32], const TO (&f)[32], const float* sa, float sw, int tokens) {
    char* o = (char*)((TO*)p.out + (size_t)m * p.ldo + n);
    const uint64_t step = (uint64_t)(uint32_t)p.ldo * sizeof(TO);
    if (tokens >= 32) {
        const float2 sw2 = make_float2(sw, sw);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const float4 s = *(const float4*)(sa + i);
#pragma unroll
            for (int j = 0; j < 4; j += 2, o += 2 * step) {
                const float2 t = f2_mul(j ? make_float2(s.z, s.w) : make_float2(s.x, s.y), sw2);
                float2 v = f2_mul(make_float2((float)(int)r[i + j], (float)(int)r[i + j + 1]), t);
                if (RES) v = make_float2(v.x + to_f32(f[i + j]), v.y + to_f32(f[i + j + 1]));
                store_pair((TO*)o, (TO*)(o + step), v);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i, o += step) {
            if (i >= tokens) break;
            const float v = (float)(int)r[i] * (sa[i] * sw);
            *(TO*)o = from_f32<TO>(RES ? v + to_f32(f[i]) : v);
        }
    }
}
// this warp's copy of a tile's token scales
__device__ __forceinline__ void load_scales(const Q8Args& p, float* sa, int m0, int lane) {
    for (int j = lane; j < p.bn; j += 32) sa[j] = m0 + j < p.M ? p.scale[m0 + j] : 0.0f;
    __syncwarp();
}

// the instructions of one k-block; the last block of K may hold fewer than four (what lies beyond K is zero)
__device__ __forceinline__ int instructions(const Q8Args& p, int kb) { return min(BK / UK, (p.K - kb * BK + UK - 1) / UK); }

// a wait ran out somewhere in this CTA: let copies and products in flight land before their memory is given back, and say so
__device__ __forceinline__ void report_abort(const Q8Args& p, volatile int* abort_flag, uint64_t grace_ns) {
    if (!*abort_flag) return;
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < grace_ns) __nanosleep(1000);
    if (threadIdx.x == 0 && p.err) atomicExch(p.err, 3000);
}

// ---- few tokens ------------------------------------------------------------------------------------------------------------------------
// A warp per channel, the lanes along K: 16 codes of every row per step, four at a time in the four-way byte product. Setting up tensor
// memory, barriers and tensor maps costs more than the whole product of one token (1 x 960 -> 1600: 3.8 us there); here a call is a round
// or two of loads and one reduction.
constexpr int FEW_WARPS = 8, FEW_TOKENS = 4;
// (No __restrict__: what the kernel in front writes must not come through the read-only path.)
template <typename TO, bool RES, int MT>
__global__ void __launch_bounds__(32 * FEW_WARPS) q8_few_kernel(const Q8Args p, const int8_t* q, int ldq, const int8_t* w) {
    const int lane = threadIdx.x & 31, n = (int)blockIdx.x * FEW_WARPS + (int)(threadIdx.x >> 5), chunks = p.K >> 4;
    const int8_t* wr = w + (size_t)min(n, p.N - 1) * p.K;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int k = lane; k < chunks; k += 32) prefetch_l2(wr + 16 * k);   // while the preceding kernel still runs
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (n >= p.N) return;
    int acc[MT] = {};
#pragma unroll 4
    for (int k = lane; k < chunks; k += 32) {
        const int4 b = *(const int4*)(wr + 16 * k);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int4 a = *(const int4*)(q + (size_t)min(m, p.M - 1) * ldq + 16 * k);
            acc[m] = __dp4a(a.x, b.x, __dp4a(a.y, b.y, __dp4a(a.z, b.z, __dp4a(a.w, b.w, acc[m]))));
        }
    }
    int mine = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int total = __reduce_add_sync(0xffffffffu, acc[m]);
        if (lane == m) mine = total;
    }
    if (lane < p.M) {   // M <= MT tokens
        const float v = (float)mine * (p.scale[lane] * p.wscale[n]);
        ((TO*)p.out)[(size_t)lane * p.ldo + n] = from_f32<TO>(RES ? v + to_f32(((const TO*)p.residual)[(size_t)lane * p.ldr + n]) : v);
    }
}

// ---- split-K over a cluster ------------------------------------------------------------------------------------------------------------
struct __align__(8) SplitBarriers {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc, sums;
    uint32_t tmem_base;
    int abort_flag;
};

template <typename TO, bool RES>
__global__ void __launch_bounds__(NUM_THREADS) q8_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmQ, const Q8Args p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ SplitBarriers bars;
    __shared__ __align__(16) float s_sa[4][256];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int b_bytes = p.bn * BK, stage_bytes = A_BYTES + b_bytes;
    int* red = (int*)(smem + p.stages * stage_bytes);   // [splits][bn / splits][128]: every CTA's partial sums of this CTA's tokens
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // uniform for the compiler, too
    const int split = p.splits > 1 ? (int)cluster_ctarank() : 0;
    const int tile = (int)blockIdx.x / p.splits;
    const int m0 = tile / p.tiles_ch * p.bn, n0 = tile % p.tiles_ch * BM;
    const int kb0 = split * p.kb_per, kb1 = min(p.kb_total, kb0 + p.kb_per);
    const uint32_t tmem_cols = p.bn <= 32 ? 32u : p.bn <= 64 ? 64u : p.bn <= 128 ? 128u : 256u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.empty[s], 1);
        }
        mbar_init(&bars.acc, 1);
        mbar_init(&bars.sums, 1);
        bars.abort_flag = 0;
        mbar_fence_init();
        if (p.splits > 1) mbar_expect_tx(&bars.sums, (uint32_t)(p.bn * BM * 4));   // this CTA's tokens from every CTA of the cluster
        fence_proxy_async_smem();
    }
    if (warp == 1) {
        tmem_alloc(&bars.tmem_base, tmem_cols);
        tmem_relinquish();
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        // Into L2 while the preceding kernel still runs: the weights (a prefetch returns nothing, so it does not matter if that kernel is the
        // one that writes them) and the two tensor maps.
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmQ);
        for (int kb = kb0; kb < kb1; ++kb) tma_prefetch_l2_2d(&tmW, kb * BK, n0);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (p.splits > 1) cluster_arrive();   // "this CTA runs and its barriers exist": waited for before the first store to a peer
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t tmem_base = bars.tmem_base;
    volatile int* abort_flag = &bars.abort_flag;
    bool ok = true;
    float sw4[4];

    if (warp == 0) {
        const bool lead = elect_one();
        for (int kb = kb0, i = 0; kb < kb1 && ok; ++kb, ++i) {
            const int s = i % p.stages;
            if (i >= p.stages) ok = __all_sync(0xffffffffu, mbar_wait(&bars.empty[s], (i / p.stages - 1) & 1, abort_flag));
            if (ok && lead) {
                uint8_t* st = smem + s * stage_bytes;
                mbar_expect_tx(&bars.full[s], (uint32_t)stage_bytes);
                tma_load_2d(st, &tmW, &bars.full[s], kb * BK, n0);
                tma_load_2d(st + A_BYTES, &tmQ, &bars.full[s], kb * BK, m0);
            }
            __syncwarp();
        }
        // the CTA may not retire while commits can still arrive on `empty`
        for (int i = max(0, kb1 - kb0 - p.stages); i < kb1 - kb0 && ok; ++i) ok = mbar_wait(&bars.empty[i % p.stages], (i / p.stages) & 1, abort_flag);
    } else if (warp == 1) {
        const bool lead = elect_one();
        const uint32_t idesc = umma_idesc_s8_s32(BM, p.bn);
        for (int kb = kb0, i = 0; kb < kb1 && ok; ++kb, ++i) {
            const int s = i % p.stages;
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.full[s], (i / p.stages) & 1, abort_flag));
            if (ok && lead) {
                tc_fence_after_sync();
                const uint32_t at = smem_u32(smem + s * stage_bytes);
                const uint64_t ad = umma_smem_desc_sw128(at, 16, 1024), bd = umma_smem_desc_sw128(at + A_BYTES, 16, 1024);
                const int n = instructions(p, kb);
                umma_s8_ss(tmem_base, ad, bd, idesc, i > 0);
#pragma unroll
                for (int k = 1; k < BK / UK; ++k)
                    if (k < n) umma_s8_ss(tmem_base, ad + 2 * k, bd + 2 * k, idesc, 1);
                umma_commit(&bars.empty[s]);
            }
            __syncwarp();
        }
        if (ok && lead) umma_commit(&bars.acc);
        __syncwarp();
    } else {
        const int qd = warp & 3, n = n0 + qd * 32 + lane;
        float* sa = s_sa[qd];
        load_scales(p, sa, m0, lane);
        const float sw = n < p.N ? p.wscale[n] : 0.0f;
        if (p.splits > 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sw4[i] = n0 + 4 * lane + i < p.N ? p.wscale[n0 + 4 * lane + i] : 0.0f;
            cluster_wait();   // here, where there is time: the products are still being made
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.acc, 0, abort_flag));
        if (ok) {
            tc_fence_after_sync();
            if (p.splits == 1)
                for (int c0 = 0; c0 < p.bn && m0 + c0 < p.M; c0 += 32) {
                    uint32_t r[32];
                    TO f[32];
                    const int tokens = min(p.bn, p.M - m0) - c0;
                    if (RES && n < p.N) load_residual<TO>(p, m0 + c0, n, f, tokens);
                    tmem_ld_32x32(tmem_base + ((uint32_t)(qd * 32) << 16) + c0, r);
                    tmem_ld_wait();
                    if (n < p.N) store_tokens<TO, RES>(p, m0 + c0, n, r, f, sa + c0, sw, tokens);
                    __syncwarp();
                }
        }
    }
    if (p.splits > 1) {
        // Every CTA finishes bn / splits of the tokens: partial sums go to their owners' shared memory by asynchronous stores, whose bytes the
        // owner's barrier counts; it adds them, a warp per token, four channels a lane.
        const int own = p.bn / p.splits, log_own = 31 - __clz(own), qd = warp & 3, n = n0 + 4 * lane;
        __syncwarp();   // the barrier instruction wants whole warps
        if (warp < 2) cluster_wait();
        if (warp >= 2 && ok) {
            for (int c0 = 0; c0 < p.bn; c0 += 32) {
                uint32_t r[32];
                tmem_ld_32x32(tmem_base + ((uint32_t)(qd * 32) << 16) + c0, r);
                tmem_ld_wait();
                const int* to = red + split * own * BM + qd * 32 + lane;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i < 16 || p.bn > 16) {
                        const uint32_t owner = (uint32_t)(c0 + i) >> log_own;
                        st_async_u32(mapa_shared(to + ((c0 + i) & (own - 1)) * BM, owner), r[i], mapa_shared(&bars.sums, owner));
                    }
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(&bars.sums, 0, abort_flag));
            for (int c = qd; c < own && ok; c += 4) {
                const int j = split * own + c, m = m0 + j;
                if (m >= p.M || n >= p.N) break;
                TO f[4];
                if (RES) {
                    const TO* res = (const TO*)p.residual + (size_t)m * p.ldr + n;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < p.N) f[i] = res[i];
                }
                int sum[4] = {};
                for (int s = 0; s < p.splits; ++s) {
                    const int4 v = *(const int4*)(red + (s * own + c) * BM + 4 * lane);
                    sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
                }
                const float sa = s_sa[qd][j];
                TO* o = (TO*)p.out + (size_t)m * p.ldo + n;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.N) {
                        const float v = (float)sum[i] * (sa * sw4[i]);
                        o[i] = from_f32<TO>(RES ? v + to_f32(f[i]) : v);
                    }
            }
        }
    }
    __syncwarp();
    report_abort(p, abort_flag, p.splits > 1 ? 2500000000ull : 2000000ull);   // a peer may still write here until its own wait has run out, too
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem_base, tmem_cols);
}

// ---- persistent CTA pairs --------------------------------------------------------------------------------------------------------------
// A pair computes 256 channels x bn tokens; K streams through a shared-memory ring, the accumulators of the next tile are filled while this
// one is stored. HELD (K of at most HELD_BLOCKS k-blocks): a tile's weights stay in shared memory while the pair walks the tokens, which halves
// the bytes of a tile. With both operands streaming, every k-block of a 256 x 256 tile brings 32 KB to each SM for 512 cycles of products; the
// L2 gives an SM 45 to 60 bytes per cycle when all of them ask, the output's bytes included (32768 x 960 -> 5120: 131 us held, 138 streamed).
// Tokens as the A operand, their rows stored in 16-byte pieces through shared memory, was slower (145 us): the products' own operand reads and
// the copies already fill most of the 128 bytes that an SM's shared memory moves per cycle.
constexpr int KPS = 2;                    // k-blocks per ring stage: one wait and one commit for eight instructions
constexpr int PAIR_STAGES = 3;
constexpr int HELD_BLOCKS = 8;
constexpr int HELD_BN = 224;              // widest token tile whose ring fits beside 128 KB of weights
constexpr int EPI_WARPS = 8;              // two per lane quarter, taking 32-token chunks in turn
constexpr int PAIR_THREADS = 96 + 32 * EPI_WARPS;   // warps 0 and 1 copy, warp 2 issues the products
// All that a CTA may ask for, whatever the ring needs: a CTA of the split kernel must not run beside one of this kernel. Both hold tensor
// memory while they wait for other CTAs of theirs; on two SMs (two streams) each could hold what the other's peer is still waiting to allocate.
// CTAs of the split kernel alone never run out: a cluster's fit an SM at most 512 / columns times by their shared memory.
constexpr int PAIR_SMEM = 222 * 1024;
constexpr int pair_ring(bool held) { return held ? HELD_BLOCKS * A_BYTES + PAIR_STAGES * KPS * (HELD_BN / 2) * BK : PAIR_STAGES * KPS * 2 * A_BYTES; }
static_assert(pair_ring(false) + 1024 <= PAIR_SMEM && pair_ring(true) + 1024 <= PAIR_SMEM, "shared memory budget");

struct __align__(8) PairBarriers {
    uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], acc_full[2], acc_empty[2], held_full, held_empty;
    uint32_t tmem_base;
    int abort_flag;
};

// The units of one pair, in order. Streaming: round-robin over the pairs; channel tiles run fastest inside groups of RASTER of them, so that
// a wave shares its tokens and one group's weights stay in L2. Held: a contiguous run of units, tokens fastest.
constexpr int RASTER = 32;
template <bool HELD> struct Units {
    int u, end, step;
    __device__ __forceinline__ Units(const Q8Args& p, int worker, int workers) {
        const int64_t all = (int64_t)p.tiles_ch * p.tiles_tok;
        u = HELD ? (int)(all * worker / workers) : worker;
        end = HELD ? (int)(all * (worker + 1) / workers) : (int)all;
        step = HELD ? 1 : workers;
    }
    __device__ __forceinline__ bool more() const { return u < end; }
    __device__ __forceinline__ void next() { u += step; }
    // first channel and token of the unit
    __device__ __forceinline__ void tile(const Q8Args& p, int& n0, int& m0) const {
        int tok, ch;
        if (HELD) {
            ch = u / p.tiles_tok;
            tok = u - ch * p.tiles_tok;
        } else {
            const int per_group = RASTER * p.tiles_tok;
            const int g = u / per_group, idx = u - g * per_group, w = min(RASTER, p.tiles_ch - g * RASTER);
            tok = idx / w;
            ch = g * RASTER + idx - tok * w;
        }
        n0 = ch * 2 * BM;
        m0 = tok * p.bn;
    }
};

template <typename TO, bool RES, bool HELD>
__global__ void __launch_bounds__(PAIR_THREADS, 1) q8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmQ, const Q8Args p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ PairBarriers bars;
    __shared__ __align__(16) float s_sa[EPI_WARPS][128];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t rank = cluster_ctarank();
    const int worker = blockIdx.x >> 1, workers = gridDim.x >> 1;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // uniform for the compiler, too
    const int half = p.bn / 2, b_bytes = half * BK;
    // HELD: [8 k-blocks of weights][ring of tokens]; otherwise a ring of [2 k-blocks of weights][2 k-blocks of tokens]
    const int st_bytes = KPS * (HELD ? b_bytes : A_BYTES + b_bytes);
    uint8_t* ring = smem + (HELD ? HELD_BLOCKS * A_BYTES : 0);
    const int b_at = HELD ? 0 : KPS * A_BYTES;

    if (threadIdx.x == 0) {
        for (int s = 0; s < PAIR_STAGES; ++s) {
            mbar_init(&bars.full[s], 2);    // the leader's is used, by its two producers; both CTAs' copies count their bytes on it
            mbar_init(&bars.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars.acc_full[b], 1);
            mbar_init(&bars.acc_empty[b], 2 * EPI_WARPS);   // the leader's collects the epilogue warps of both CTAs
        }
        mbar_init(&bars.held_full, 2);
        mbar_init(&bars.held_empty, 1);
        bars.abort_flag = 0;
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    if (warp == 2) {
        tmem_alloc_pair(&bars.tmem_base, 512);
        tmem_relinquish_pair();
    }
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmQ);
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers exist before anything is signalled across the pair
    tc_fence_after_sync();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t tmem_base = bars.tmem_base;
    volatile int* abort_flag = &bars.abort_flag;

    if (warp == 0 || warp == 1) {
        // Producer `warp` brings the first or second k-block of every stage (a copy costs its issuing thread 100 to 200 cycles: one thread
        // for all of them was half as long as the products they feed).
        const int j = warp;
        const bool lead = elect_one();
        int s = 0, held = -1, loads = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (Units<HELD> it(p, worker, workers); it.more() && ok; it.next()) {
            int m0, n0;
            it.tile(p, n0, m0);
            if (HELD && n0 != held) {
                // other weights: once the products with the ones held so far have been made
                if (loads > 0) {
                    ok = mbar_wait(&bars.held_empty, (loads - 1) & 1, abort_flag);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                }
                if (lead) {
                    const uint32_t full = mapa_shared(&bars.held_full, 0);
                    if (rank == 0) mbar_expect_tx(&bars.held_full, (uint32_t)(2 * ((p.kb_total + 1 - j) / 2) * A_BYTES));
                    for (int kb = j; kb < p.kb_total; kb += 2) tma_load_2d_pair(smem + kb * A_BYTES, &tmW, full, kb * BK, n0 + (int)rank * BM);
                }
                __syncwarp();
                held = n0;
                ++loads;
            }
            n0 += (int)rank * BM;
            m0 += (int)rank * half;
            for (int kb = j; kb < p.kb_total + j; kb += KPS, s = (s + 1 == PAIR_STAGES ? 0 : s + 1), ph ^= (s == 0)) {
                ok = mbar_wait(&bars.empty[s], ph ^ 1, abort_flag);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                if (lead) {
                    const bool some = kb < p.kb_total;   // the second half of a tile's last stage may be empty
                    uint8_t* st = ring + s * st_bytes;
                    const uint32_t full = mapa_shared(&bars.full[s], 0);
                    if (rank == 0) mbar_expect_tx(&bars.full[s], some ? (uint32_t)(2 * ((HELD ? 0 : A_BYTES) + b_bytes)) : 0u);
                    if (some) {
                        if (!HELD) tma_load_2d_pair(st + j * A_BYTES, &tmW, full, kb * BK, n0);
                        tma_load_2d_pair(st + b_at + j * b_bytes, &tmQ, full, kb * BK, m0);
                    }
                }
                __syncwarp();
            }
        }
        // the CTA may not retire while commits can still arrive on its barriers
        for (int i = 0; i < PAIR_STAGES && ok; ++i, s = (s + 1 == PAIR_STAGES ? 0 : s + 1), ph ^= (s == 0))
            if (!mbar_wait(&bars.empty[s], ph ^ 1, abort_flag)) ok = false;
    } else if (warp == 2) {
        // The whole warp runs the loop and one elected lane issues: with warp-uniform descriptors an instruction costs the issuing warp 40
        // cycles instead of 48. Whole stages are straight code; only the last stage of a tile counts its instructions.
        if (rank == 0) {
            const bool lead = elect_one();
            const uint32_t idesc = umma_idesc_s8_s32(2 * BM, p.bn);
            const uint64_t ad0 = umma_smem_desc_sw128(smem_u32(smem), 16, 1024), bd0 = umma_smem_desc_sw128(smem_u32(ring + b_at), 16, 1024);
            const uint32_t st16 = (uint32_t)st_bytes >> 4, b16 = (uint32_t)b_bytes >> 4;
            const int last_kb = (p.kb_total - 1) / KPS * KPS;                       // first k-block of the last stage
            const int last_n = (p.K - last_kb * BK + UK - 1) / UK;                  // its instructions, 1 to 8
            int s = 0, i = 0, held = -1, loads = 0;
            uint32_t ph = 0, off = 0;
            bool ok = true;
            for (Units<HELD> it(p, worker, workers); it.more() && ok; it.next(), ++i) {
                const int buf = i & 1;
                if (HELD) {
                    int m0, n0;
                    it.tile(p, n0, m0);
                    if (n0 != held) {
                        if (loads > 0 && lead) umma_commit_pair(&bars.held_empty, 3);   // behind the last product with the previous weights
                        ok = mbar_wait(&bars.held_full, loads & 1, abort_flag);
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                        held = n0;
                        ++loads;
                    }
                }
                ok = mbar_wait(&bars.acc_empty[buf], ((i >> 1) & 1) ^ 1, abort_flag);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t d = tmem_base + buf * 256;
                for (int kb = 0; kb < p.kb_total; kb += KPS) {
                    ok = mbar_wait(&bars.full[s], ph, abort_flag);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint64_t ad = ad0 + (HELD ? (uint32_t)kb * (A_BYTES >> 4) : off), bd = bd0 + off, bd1 = bd + b16;
                    if (lead) {
                        const int n = kb == last_kb ? last_n : 8;
                        umma_s8_ss_pair(d, ad, bd, idesc, kb > 0);
                        if (n == 8) {
#pragma unroll
                            for (int k = 1; k < 4; ++k) umma_s8_ss_pair(d, ad + 2 * k, bd + 2 * k, idesc, 1);
#pragma unroll
                            for (int k = 0; k < 4; ++k) umma_s8_ss_pair(d, ad + (A_BYTES >> 4) + 2 * k, bd1 + 2 * k, idesc, 1);
                        } else {
#pragma unroll
                            for (int k = 1; k < 7; ++k)
                                if (k < n) umma_s8_ss_pair(d, ad + (k >> 2) * (A_BYTES >> 4) + 2 * (k & 3), (k < 4 ? bd : bd1) + 2 * (k & 3), idesc, 1);
                        }
                        umma_commit_pair(&bars.empty[s], 3);
                    }
                    __syncwarp();
                    if (++s == PAIR_STAGES) { s = 0; ph ^= 1u; off = 0; }
                    else off += st16;
                }
                if (ok && lead) umma_commit_pair(&bars.acc_full[buf], 3);
                __syncwarp();
            }
        }
    } else {
        // Two warps per lane quarter take the 32-token chunks of a tile in turn. A tile's scales are loaded while the tile before is stored, a
        // chunk's residual while the chunk before is: loaded when they are needed, their latency was a third of the epilogue and more.
        const int qd = warp & 3, e = warp - 3, first = (e >> 2) * 32;
        float* sa = s_sa[e];
        float next_sa[4], next_sw = 0.0f;
        const auto fetch = [&](const Units<HELD>& it) {
            int m0, n0;
            it.tile(p, n0, m0);
            const int n = n0 + (int)rank * BM + qd * 32 + lane;
            next_sw = n < p.N ? p.wscale[n] : 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = first + 64 * k + lane;
                next_sa[k] = c < p.bn && m0 + c < p.M ? p.scale[m0 + c] : 0.0f;
            }
        };
        Units<HELD> it(p, worker, workers);
        if (it.more()) fetch(it);
        for (int i = 0; it.more(); ++i) {
            int m0, n0;
            it.tile(p, n0, m0);
            const int buf = i & 1, n = n0 + (int)rank * BM + qd * 32 + lane;
            const float sw = next_sw;
#pragma unroll
            for (int k = 0; k < 4; ++k) sa[32 * k + lane] = next_sa[k];
            __syncwarp();
            it.next();
            if (it.more()) fetch(it);
            const uint32_t t0 = tmem_base + ((uint32_t)(qd * 32) << 16) + (uint32_t)(buf * 256);
            const uint32_t done = mapa_shared(&bars.acc_empty[buf], 0);
            const float* s = sa;
            const int stop = min(p.bn, p.M - m0);
            TO res[32];
            if (RES && n < p.N) load_residual<TO>(p, m0 + first, n, res, stop - first);
            if (!__all_sync(0xffffffffu, mbar_wait(&bars.acc_full[buf], (i >> 1) & 1, abort_flag))) break;
            tc_fence_after_sync();
            for (int c0 = first; c0 < stop; c0 += 64, s += 32) {
                uint32_t r[32];
                tmem_ld_32x32(t0 + c0, r);
                tmem_ld_wait();
                if (c0 + 64 >= stop) {   // the accumulator has been read: the next tile but one may have it while this one is stored
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster_relaxed(done);
                }
                if (n < p.N) {
                    TO f[32];
                    if (RES) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] = res[j];
                        load_residual<TO>(p, m0 + c0 + 64, n, res, stop - c0 - 64);
                    }
                    store_tokens<TO, RES>(p, m0 + c0, n, r, f, s, sw, stop - c0);
                }
                __syncwarp();
            }
            if (first >= stop && lane == 0) mbar_arrive_cluster_relaxed(done);   // a last tile without a chunk for this warp
        }
    }
    __syncwarp();
    report_abort(p, abort_flag, 2000000ull);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // no signal of the peer may still be on its way to this CTA's barriers
    tc_fence_after_sync();
    if (warp == 2) tmem_dealloc_pair(tmem_base, 512);
}

// ---- launch ----------------------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// codes[rows][K] at a pitch of `ld` bytes, in boxes of box_rows rows x one k-block, 128-byte swizzle, zeros outside
bool code_map(CUtensorMap* tm, const void* base, int K, int rows, int64_t ld, int box_rows) {
    static const EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (EncodeTiledFn)f : nullptr;
    }();
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {BK, (cuuint32_t)box_rows}, step[2] = {1, 1};
    return fn && fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int ceil_div(int a, int b) { return a / b + (a % b != 0); }

constexpr int SPLIT_RING = 96 * 1024;   // two CTAs of the split kernel fit on an SM
int split_stages(int bn, int kb_per) {
    const int fit = SPLIT_RING / (A_BYTES + bn * BK);
    return std::min(std::min(fit, MAX_STAGES), kb_per);
}
int split_smem(int bn, int splits, int kb_per) { return split_stages(bn, kb_per) * (A_BYTES + bn * BK) + (splits > 1 ? bn * BM * 4 : 0) + 1024; }

enum { Q8_PAIR, Q8_HELD, Q8_SPLIT, Q8_FEW };
struct Plan {
    int kind, bn, splits;
};

// The estimated time, in microseconds, of every kernel and tile that can take the product; the smallest is taken. The constants were fitted to
// 663 products (1 to 32768 tokens, K 128 to 11008, 576 to 14336 channels, both types, with and without a residual) that were timed with every
// plan: the plan taken is 1.2 % slower than the best one in the mean and 27 % at the most (K = 128 with a residual). What the terms stand for,
// with the bytes of a k-block at the rate that an SM gets from L2:
//   split  2.1 of launch and set-up, more for the exchange over a cluster; per CTA a k-block is its bytes, or the 0.32 that its issuing threads
//          need, and a token its stores; two CTAs share an SM where their shared memory allows, and then run at half the speed each
//   pair   2.3; per tile and k-block the bytes, the products or the issuing threads; the stores of a tile share the path to L2 with the next
//          tile's loads. Held weights: no bytes for them, but they are loaded before the first product.
//   few    one to four tokens: the weights' bytes, and the tokens' codes from L1 once per step of 2048 codes
Plan choose(int M, int N, int K, int sms) {
    const int kb = ceil_div(K, BK);
    Plan best{Q8_SPLIT, 16, 1};
    double least = 1e30;
    const auto offer = [&](double t, Plan plan) {
        if (t < least) { least = t; best = plan; }
    };
    for (int bn = 16; bn <= 256 && (bn == 16 || bn / 2 < M); bn *= 2)
        for (int s = 1; s <= (bn <= 128 ? 8 : 1); s *= 2) {
            const int per = ceil_div(kb, s);
            if ((s - 1) * per >= kb) continue;   // a CTA without a k-block
            const double ctas = (double)ceil_div(N, BM) * ceil_div(M, bn) * s;
            const bool two = split_smem(bn, s, per) <= 112 * 1024;
            const double rounds = two && ctas <= 2 * sms ? std::max(1.0, ctas / sms) : std::ceil(ctas / sms);
            offer(2.1 + (s > 1 ? 0.16 + 0.044 * bn : 0.0) + rounds * (per * std::max((A_BYTES + bn * BK) * 1.6e-5, 0.32) + 0.0073 * bn / s), Plan{Q8_SPLIT, bn, s});
        }
    for (int kind = Q8_PAIR; kind <= (kb <= HELD_BLOCKS ? Q8_HELD : Q8_PAIR); ++kind)
        for (int bn = 64; bn <= (kind == Q8_HELD ? HELD_BN : 256) && (bn == 64 || bn / 2 < M); bn += 32) {
            const double rounds = std::ceil((double)ceil_div(N, 2 * BM) * ceil_div(M, bn) / (sms / 2));
            const double block = std::max({((kind == Q8_HELD ? 0 : A_BYTES) + bn / 2 * BK) * 8.1e-6, 8.8e-4 * bn, 0.21});
            offer(2.3 + (kind == Q8_HELD ? 0.23 * kb : 0.0) + rounds * (kb * block + 0.0052 * bn), Plan{kind, bn, 1});
        }
    if (M <= FEW_TOKENS) offer(0.11 + 0.41 * ceil_div(K, 2048) * (1 + M) + (1.1e-7 + 1.5e-8 * M) * K * N, Plan{Q8_FEW, M, 1});
    return best;
}

template <typename TO, bool RES> int launch(Q8Args p, const int8_t* q, int ldq, const int8_t* w, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    const int rc = set_up_once(done, [] {
        const auto allow = [](auto* kernel, int bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess; };
        return allow(q8_pair_kernel<TO, RES, false>, PAIR_SMEM) && allow(q8_pair_kernel<TO, RES, true>, PAIR_SMEM) &&
               allow(q8_split_kernel<TO, RES>, split_smem(128, 2, MAX_STAGES)) ? 0 : -5;
    });
    if (rc) return rc;
    const int sms = sm_count_current_device();
    const Plan plan = choose(p.M, p.N, p.K, sms);
    static const bool overlap = getenv("BM_NO_PDL") == nullptr;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = overlap ? 2 : 1;
    if (plan.kind == Q8_FEW) {
        using Kernel = void (*)(Q8Args, const int8_t*, int, const int8_t*);
        const Kernel few = p.M == 1 ? (Kernel)q8_few_kernel<TO, RES, 1> : p.M == 2 ? (Kernel)q8_few_kernel<TO, RES, 2> : (Kernel)q8_few_kernel<TO, RES, FEW_TOKENS>;
        at[0] = at[1];
        cfg.numAttrs = overlap ? 1 : 0;
        cfg.blockDim = dim3(32 * FEW_WARPS);
        cfg.gridDim = dim3((unsigned)ceil_div(p.N, FEW_WARPS));
        if (cudaLaunchKernelEx(&cfg, few, p, q, ldq, w) == cudaSuccess) return 0;
        cudaGetLastError();
        return -9;
    }
    CUtensorMap tmW, tmQ;
    p.bn = plan.bn;
    p.kb_total = ceil_div(p.K, BK);
    p.tiles_tok = ceil_div(p.M, plan.bn);
    p.tiles_ch = ceil_div(p.N, plan.kind == Q8_SPLIT ? BM : 2 * BM);
    if (!code_map(&tmW, w, p.K, p.N, p.K, BM) || !code_map(&tmQ, q, p.K, p.M, ldq, plan.kind == Q8_SPLIT ? plan.bn : plan.bn / 2)) return -11;
    const int64_t tiles = (int64_t)p.tiles_ch * p.tiles_tok;
    cudaError_t e;
    if (plan.kind != Q8_SPLIT) {
        if (tiles > 0x3fffffff) return -1;
        at[0].val.clusterDim.x = 2;
        cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, sms / 2)));
        cfg.blockDim = dim3(PAIR_THREADS);
        cfg.dynamicSmemBytes = PAIR_SMEM;
        e = cudaLaunchKernelEx(&cfg, plan.kind == Q8_HELD ? q8_pair_kernel<TO, RES, true> : q8_pair_kernel<TO, RES, false>, tmW, tmQ, p);
    } else {
        if (tiles * plan.splits > 0x7fffffff) return -1;
        p.splits = plan.splits;
        p.kb_per = ceil_div(p.kb_total, plan.splits);
        p.stages = split_stages(plan.bn, p.kb_per);
        at[0].val.clusterDim.x = (unsigned)plan.splits;
        cfg.gridDim = dim3((unsigned)(tiles * plan.splits));
        cfg.dynamicSmemBytes = (size_t)split_smem(plan.bn, plan.splits, p.kb_per);
        e = cudaLaunchKernelEx(&cfg, q8_split_kernel<TO, RES>, tmW, tmQ, p);
    }
    if (e == cudaSuccess) return 0;
    cudaGetLastError();   // a launch that failed must not poison the status of later calls
    return -9;
}

}  // namespace

int q8_matmul(int dtype, void* out, int ldo, const int8_t* q, int ldq, const float* scale, const int8_t* w, const float* wscale, const void* residual,
              int ldr, int M, int K, int N, int* err, cudaStream_t st) {
    if (M > 0x7fffff00 || N > 0x7fffff00) return -1;   // tile origins are 32-bit
    Q8Args p = {};
    p.out = out; p.residual = residual; p.scale = scale; p.wscale = wscale;
    p.ldo = ldo; p.ldr = ldr; p.M = M; p.N = N; p.K = K; p.err = err;
    if (dtype) return residual ? launch<bf16, true>(p, q, ldq, w, st) : launch<bf16, false>(p, q, ldq, w, st);
    return residual ? launch<float, true>(p, q, ldq, w, st) : launch<float, false>(p, q, ldq, w, st);
}

}  // namespace bmb
