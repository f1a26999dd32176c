// yolo_linear: y = act(x W^T + b) + r for row-major x [M,K], W [N,K] (both contiguous in K), the 1x1 convolution of
// conv2d (reference yolo_v3/utils/layer_utils.py:9-21) for weights that live in the caller's device memory, with the
// residual added after the activation like res_block (layer_utils.py:24-29).
//
// Mathematics: one matrix product with f32 accumulators on MFMA, bias / activation / residual applied to the accumulators,
// ONE rounding to the storage type at the store.  2MNK operations over (M+N)K elements read and MN written (2MN with r).
#include <type_traits>

#include "layer_common.h"

namespace yolo {

struct LinK {
    const char* x;
    const char* w;
    const void* bias;
    const char* res;
    char* out;
    long long x_ld, w_ld, res_ld, out_ld;   // bytes per row
    long long M;
    int N, K;
    int bias_bf16, act;
    int vec_out;                            // out / residual rows are 16-byte aligned
    unsigned ntm, ntn;
};

// gelu(v) = v * Phi(v) = v/2 * erfc(-v / sqrt 2).  f32 results take the library's erfcf (no cancellation in the negative tail);
// for bf16 results erfc(z), z >= 0, is Abramowitz & Stegun 7.1.26 (|error| <= 1.5e-7, a bf16 half step is 2^-9 of the value):
// one reciprocal, one exponential and six multiply-adds against about forty instructions and a divergent branch, which at
// 23104 x 4096 results cost as much time as a half of the product itself.
template <bool BF16>
__device__ __forceinline__ float gelu(float v) {
    if constexpr (!BF16) {
        return 0.5f * v * erfcf(-0.70710678118654752f * v);
    } else {
        const float z = __builtin_fabsf(v) * 0.70710678118654752f;
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, z, 1.0f));
        float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
        p = __builtin_fmaf(p, t, 1.421413741f);
        p = __builtin_fmaf(p, t, -0.284496736f);
        p = __builtin_fmaf(p, t, 0.254829592f);
        const float e = p * t * __builtin_amdgcn_exp2f(z * z * -1.4426950408889634f);      // erfc(z)
        return 0.5f * v * (v < 0.f ? e : 2.0f - e);
    }
}

template <bool BF16, int ACT>
__device__ __forceinline__ float activate(float v) {
    if constexpr (ACT == YOLO_ACT_LEAKY) return v > 0.f ? v : 0.1f * v;
    else if constexpr (ACT == YOLO_ACT_RELU) return v < 0.f ? 0.f : v;
    else if constexpr (ACT == YOLO_ACT_GELU) return gelu<BF16>(v);
    else if constexpr (ACT == YOLO_ACT_SILU) {
        if constexpr (BF16) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
        else return v / (1.0f + expf(-v));
    } else return v;
}

// Calls f(integral_constant<int, ACT>) for the runtime activation, so that element loops hold no branch.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
        case YOLO_ACT_LEAKY: f(std::integral_constant<int, YOLO_ACT_LEAKY>{}); break;
        case YOLO_ACT_RELU: f(std::integral_constant<int, YOLO_ACT_RELU>{}); break;
        case YOLO_ACT_GELU: f(std::integral_constant<int, YOLO_ACT_GELU>{}); break;
        case YOLO_ACT_SILU: f(std::integral_constant<int, YOLO_ACT_SILU>{}); break;
        default: f(std::integral_constant<int, YOLO_ACT_NONE>{}); break;
    }
}

// One 64-byte K-slice of 16 rows against 16 rows: lane l holds the 16-byte piece (l / 16) of row l % 16 of either operand.
// bf16: one 16x16x32 MFMA.  f32: four 16x16x4, MFMA j takes element j of every lane's piece (the four k of an MFMA are 4 apart,
// the same in both operands, so every k meets its partner once).  Accumulator: lane l, register r = D[4 * (l / 16) + r][l % 16].
template <bool BF16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[j], fb[j], c, 0, 0, 0);
        return c;
    }
}

// The 16-byte piece of a row that starts at element k, elements past K as zeros.  Rows need no alignment beyond their element's:
// a whole piece is one load (global memory takes any address), the last one goes element by element.
template <bool BF16>
__device__ __forceinline__ u32x4 load_piece(const char* row, int k, int K) {
    typedef typename Elem<BF16>::type T;
    constexpr int P = Elem<BF16>::kPiece;
    u32x4 v = {0, 0, 0, 0};
    const T* p = (const T*)row + k;
    if (k + P <= K) {
        __builtin_memcpy(&v, p, 16);
    } else {
        typename std::conditional<BF16, bf16x8, f32x4>::type e = {};
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (k + j < K) e[j] = p[j];
        v = __builtin_bit_cast(u32x4, e);
    }
    return v;
}

// ---- tiles of BM rows of x by BN rows of W through LDS ------------------------------------------------------------------------
// WR x WC waves, each (BM / WR) x (BN / WC); K in steps of 128 bytes, two LDS buffers, one barrier a step: the loads of step
// s + 1 are issued before the products of step s.  An LDS row is 128 bytes = 8 pieces, piece c of row r at slot c ^ (r & 7),
// so that the 16 rows a fragment read touches fall on all banks.  W is the MFMA's first operand: a lane then holds four
// consecutive outputs of one row of y.
// ALIGNED: rows of x and W start on 16 bytes and K is whole pieces; they go global -> LDS by DMA, out-of-range rows and pieces
// read `zero` instead.  Otherwise the pieces pass through registers.
__device__ const u32x4 kZeroPiece = {0, 0, 0, 0};

template <bool BF16, int BM, int BN, int WR, int WC, bool ALIGNED>
__global__ __launch_bounds__(WR* WC * 64) void linear_tile_kernel(LinK p) {
    typedef typename Elem<BF16>::type T;
    constexpr int NT = WR * WC * 64, P = Elem<BF16>::kPiece, BK = 8 * P;
    constexpr int TM = BM / WR / 16, TN = BN / WC / 16;
    constexpr int LPT = (BM + BN) * 8 / NT;                 // pieces a thread stages per step
    constexpr int BUF = (BM + BN) * 128;
    static_assert((BM + BN) * 8 % NT == 0 && BM * 8 % NT == 0, "whole pieces per thread");
    static_assert(TN % 2 == 0, "bf16 stores pair two column tiles");
    extern __shared__ char lds[];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned tile = xcd_chunk(blockIdx.x, p.ntm * p.ntn);
    const unsigned tn = tile % p.ntn, tm = tile / p.ntn;
    const long long m0 = (long long)tm * BM;
    const int n0 = (int)tn * BN;
    const int nsteps = (p.K + BK - 1) / BK;

    const char* src[LPT];                                   // row of piece i (nullptr: past the last row)
    int kc;                                                 // element offset of this thread's pieces inside a step
    {
        const int r = tid >> 3;
        kc = ((tid & 7) ^ (r & 7)) * P;                     // NT / 8 is a multiple of 8: the same for all i
#pragma unroll
        for (int i = 0; i < LPT; ++i) {
            const int row = i * (NT / 8) + r;
            if (row < BM) src[i] = m0 + row < p.M ? p.x + (m0 + row) * p.x_ld : nullptr;
            else src[i] = n0 + row - BM < p.N ? p.w + (long long)(n0 + row - BM) * p.w_ld : nullptr;
        }
    }
    u32x4 stage[ALIGNED ? 1 : LPT];
    auto issue = [&](int s, int buf) {
        const int k = s * BK + kc;
#pragma unroll
        for (int i = 0; i < LPT; ++i) {
            if constexpr (ALIGNED) {
                const bool in = src[i] != nullptr && k < p.K;
                dma16(in ? (const void*)(src[i] + (long long)k * sizeof(T)) : (const void*)&kZeroPiece,
                      lds + buf * BUF + (i * NT + wave * 64) * 16);
            } else {
                stage[i] = u32x4{0, 0, 0, 0};
                if (src[i] != nullptr && k < p.K) stage[i] = load_piece<BF16>(src[i], k, p.K);
            }
        }
    };
    auto settle = [&](int buf) {                            // not ALIGNED: registers -> LDS
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < LPT; ++i) *(u32x4*)(lds + buf * BUF + (i * NT + tid) * 16) = stage[i];
        }
    };

    const int fr = lane & 15, fh = lane >> 4;
    const int wm0 = (wave / WC) * (BM / WR), wn0 = (wave % WC) * (BN / WC);
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    issue(0, 0);
    settle(0);
    for (int s = 0; s < nsteps; ++s) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (s + 1 < nsteps) issue(s + 1, (s + 1) & 1);
        const char* bx = lds + (s & 1) * BUF;
        const char* bw = bx + BM * 128;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int slot = ((ks * 4 + fh) ^ (fr & 7)) * 16;
            u32x4 fx[TM], fw[TN];
#pragma unroll
            for (int j = 0; j < TM; ++j) fx[j] = *(const u32x4*)(bx + (wm0 + j * 16 + fr) * 128 + slot);
#pragma unroll
            for (int i = 0; i < TN; ++i) fw[i] = *(const u32x4*)(bw + (wn0 + i * 16 + fr) * 128 + slot);
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = mma<BF16>(fw[i], fx[j], acc[i][j]);
        }
        if (s + 1 < nsteps) settle((s + 1) & 1);
    }

    // epilogue in registers: lane holds y[m][n .. n+3] for m = wm0 + 16 j + fr, n = wn0 + 16 i + 4 fh
    with_act(p.act, [&](auto mode) {
        constexpr int ACT = decltype(mode)::value;
#pragma unroll
        for (int i = 0; i < TN; i += 2) {
            f32x4 b0 = {0.f, 0.f, 0.f, 0.f}, b1 = {0.f, 0.f, 0.f, 0.f};
            const int n = n0 + wn0 + i * 16 + fh * 4;
            if (p.bias) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (n + r < p.N) b0[r] = load_param(p.bias, p.bias_bf16, n + r);
                    if (n + 16 + r < p.N) b1[r] = load_param(p.bias, p.bias_bf16, n + 16 + r);
                }
            }
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const long long m = m0 + wm0 + j * 16 + fr;
                f32x4 v0, v1;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v0[r] = activate<BF16, ACT>(acc[i][j][r] + b0[r]);
                    v1[r] = activate<BF16, ACT>(acc[i + 1][j][r] + b1[r]);
                }
                if constexpr (BF16) {
                    // v_permlane16_swap pairs the two column tiles: lane row fh then holds 8 consecutive outputs,
                    // tile i + (fh & 1), columns 8 * (fh >> 1) .. + 7, and stores 16 bytes
                    float o[8];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(v0[r]), __float_as_uint(v1[r]), false, false);
                        o[r] = __uint_as_float(sw[0]);
                        o[4 + r] = __uint_as_float(sw[1]);
                    }
                    const int nn = n0 + wn0 + (i + (fh & 1)) * 16 + (fh >> 1) * 8;
                    if (m < p.M && nn < p.N) {
                        char* orow = p.out + m * p.out_ld + (long long)nn * 2;
                        const char* rrow = p.res ? p.res + m * p.res_ld + (long long)nn * 2 : nullptr;
                        if (p.vec_out && nn + 8 <= p.N) {
                            if (rrow) {
                                const u32x4 rv = *(const u32x4*)rrow;
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    o[2 * q] += bf16_lo(rv[q]);
                                    o[2 * q + 1] += bf16_hi(rv[q]);
                                }
                            }
                            u32x4 ov;
#pragma unroll
                            for (int q = 0; q < 4; ++q) ov[q] = pack_bf16(o[2 * q], o[2 * q + 1]);
                            *(u32x4*)orow = ov;
                        } else {
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                if (nn + q < p.N)
                                    ((__bf16*)orow)[q] = (__bf16)(rrow ? o[q] + (float)((const __bf16*)rrow)[q] : o[q]);
                        }
                    }
                } else {
                    if (m < p.M) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            f32x4 v = h ? v1 : v0;
                            const int nn = n + 16 * h;
                            if (nn >= p.N) continue;
                            char* orow = p.out + m * p.out_ld + (long long)nn * 4;
                            const char* rrow = p.res ? p.res + m * p.res_ld + (long long)nn * 4 : nullptr;
                            if (p.vec_out && nn + 4 <= p.N) {
                                if (rrow) v += *(const f32x4*)rrow;
                                *(f32x4*)orow = v;
                            } else {
#pragma unroll
                                for (int q = 0; q < 4; ++q)
                                    if (nn + q < p.N) ((float*)orow)[q] = rrow ? v[q] + ((const float*)rrow)[q] : v[q];
                            }
                        }
                    }
                }
            }
        }
    });
}

// ---- few outputs: no LDS staging, K split over the waves of a workgroup ----------------------------------------------------------
// A workgroup owns 16 TM rows of x by 16 TN rows of W; its 8 waves take the 64-byte K-slices in turn, straight from memory to
// MFMA operand registers (an operand row is used by one wave only, so LDS would add a trip and save nothing), and the eight
// partial sums meet in LDS, added in wave order.  For calls whose tiles would leave most CUs idle: the chain of K-steps of one
// wave is an eighth as long and every load of a wave is in flight at once.
template <bool BF16, int TM, int TN, bool ALIGNED>
__global__ __launch_bounds__(512) void linear_direct_kernel(LinK p) {
    typedef typename Elem<BF16>::type T;
    constexpr int W = 8, P = Elem<BF16>::kPiece, BK = 4 * P, BM = TM * 16, BN = TN * 16;
    __shared__ float part[W][BM * BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned tile = xcd_chunk(blockIdx.x, p.ntm * p.ntn);
    const unsigned tm = tile % p.ntm, tn = tile / p.ntm;     // row tiles of one W tile next to each other
    const long long m0 = (long long)tm * BM;
    const int n0 = (int)tn * BN;
    const int fr = lane & 15, fh = lane >> 4;
    const int nslices = (p.K + BK - 1) / BK;
    const char* xr[TM];
    const char* wr[TN];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const long long m = m0 + j * 16 + fr;
        xr[j] = m < p.M ? p.x + m * p.x_ld : nullptr;
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const int n = n0 + i * 16 + fr;
        wr[i] = n < p.N ? p.w + (long long)n * p.w_ld : nullptr;
    }
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto piece = [&](const char* row, int k) {
        const bool in = row != nullptr && k < p.K;
        if constexpr (ALIGNED) return *(in ? (const u32x4*)(row + (long long)k * sizeof(T)) : &kZeroPiece);
        else return in ? load_piece<BF16>(row, k, p.K) : u32x4{0, 0, 0, 0};
    };
    constexpr int U = 4;                                     // slices in flight; those past K read zeros
    for (int s = wave; s < nslices; s += U * W) {
        u32x4 fx[U][TM], fw[U][TN];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (s + u * W) * BK + fh * P;
#pragma unroll
            for (int i = 0; i < TN; ++i) fw[u][i] = piece(wr[i], k);
#pragma unroll
            for (int j = 0; j < TM; ++j) fx[u][j] = piece(xr[j], k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = mma<BF16>(fw[u][i], fx[u][j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) *(f32x4*)&part[wave][(j * 16 + fr) * BN + i * 16 + fh * 4] = acc[i][j];
    __syncthreads();
    with_act(p.act, [&](auto mode) {
        constexpr int ACT = decltype(mode)::value;
        for (int e = tid; e < BM * BN; e += 512) {
            const long long m = m0 + e / BN;
            const int n = n0 + e % BN;
            if (m >= p.M || n >= p.N) continue;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v += part[w][e];
            if (p.bias) v += load_param(p.bias, p.bias_bf16, n);
            v = activate<BF16, ACT>(v);
            if (p.res) v += load_f32((const T*)(p.res + m * p.res_ld) + n);
            ((T*)(p.out + m * p.out_ld))[n] = (T)v;
        }
    });
}

template <bool BF16, int BM, int BN, int WR, int WC, bool ALIGNED>
static int launch_tile(LinK k, hipStream_t stream) {
    constexpr int kLds = 2 * (BM + BN) * 128;
    const unsigned long long ntm = (k.M + BM - 1) / BM, ntn = (k.N + BN - 1) / BN;
    YOLO_REQUIRE(ntm * ntn < (1ull << 31), YOLO_ERR_UNSUPPORTED, "linear: more than 2^31 tiles");
    k.ntm = (unsigned)ntm;
    k.ntn = (unsigned)ntn;
    if (kLds > 64 * 1024) {
        static std::atomic<bool> attr_done[16];   // setting the attribute twice is harmless, the flag only must not tear
        int dev = 0;
        YOLO_HIP_CHECK(hipGetDevice(&dev));
        if (dev >= 16 || !attr_done[dev]) {
            YOLO_HIP_CHECK(hipFuncSetAttribute((const void*)linear_tile_kernel<BF16, BM, BN, WR, WC, ALIGNED>,
                                               hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
            if (dev < 16) attr_done[dev] = true;
        }
    }
    hipLaunchKernelGGL((linear_tile_kernel<BF16, BM, BN, WR, WC, ALIGNED>), dim3(k.ntm * k.ntn), dim3(WR * WC * 64), kLds, stream, k);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}

template <bool BF16, int TM, int TN, bool ALIGNED>
static int launch_direct(LinK k, hipStream_t stream) {
    const unsigned long long ntm = (k.M + TM * 16 - 1) / (TM * 16), ntn = (k.N + TN * 16 - 1) / (TN * 16);
    YOLO_REQUIRE(ntm * ntn < (1ull << 31), YOLO_ERR_UNSUPPORTED, "linear: more than 2^31 tiles");
    k.ntm = (unsigned)ntm;
    k.ntn = (unsigned)ntn;
    hipLaunchKernelGGL((linear_direct_kernel<BF16, TM, TN, ALIGNED>), dim3(k.ntm * k.ntn), dim3(512), 0, stream, k);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}

template <bool BF16>
static int launch_linear(const LinK& k, bool aligned, hipStream_t stream) {
    const unsigned long long t128 = (unsigned long long)((k.M + 127) / 128) * ((k.N + 127) / 128);
    if (k.M <= 16) return aligned ? launch_direct<BF16, 1, 1, true>(k, stream) : launch_direct<BF16, 1, 1, false>(k, stream);
    if (t128 < 64) return aligned ? launch_direct<BF16, 2, 2, true>(k, stream) : launch_direct<BF16, 2, 2, false>(k, stream);
    if (aligned) return launch_tile<BF16, 128, 128, 2, 2, true>(k, stream);
    return launch_tile<BF16, 128, 128, 2, 2, false>(k, stream);
}

}  // namespace yolo

extern "C" int yolo_linear(int dtype, const void* x, int64_t x_ld, const void* weight, int64_t weight_ld, const void* bias,
                           int bias_dtype, const void* residual, int64_t residual_ld, void* out, int64_t out_ld, int64_t M,
                           int N, int K, int activation, void* stream) {
    using namespace yolo;
    YOLO_REQUIRE(dtype == YOLO_DTYPE_F32 || dtype == YOLO_DTYPE_BF16, YOLO_ERR_ARG, "linear: unknown dtype %d", dtype);
    YOLO_REQUIRE(bias_dtype == YOLO_DTYPE_F32 || bias_dtype == YOLO_DTYPE_BF16, YOLO_ERR_ARG, "linear: unknown bias dtype %d", bias_dtype);
    YOLO_REQUIRE(activation >= YOLO_ACT_NONE && activation <= YOLO_ACT_SILU, YOLO_ERR_ARG, "linear: unknown activation %d", activation);
    YOLO_REQUIRE(M >= 0 && N > 0 && K > 0, YOLO_ERR_ARG, "linear: bad size M=%lld N=%d K=%d", (long long)M, N, K);
    if (M == 0) return YOLO_OK;
    YOLO_REQUIRE(x && weight && out, YOLO_ERR_ARG, "linear: null pointer");
    YOLO_REQUIRE(x_ld >= K && weight_ld >= K && out_ld >= N && (!residual || residual_ld >= N), YOLO_ERR_ARG,
                 "linear: a row stride is shorter than its row");
    YOLO_REQUIRE(N <= (1 << 30) && K <= (1 << 30) && M <= (1ll << 40), YOLO_ERR_UNSUPPORTED, "linear: N, K <= 2^30, M <= 2^40");
    const int z = dtype == YOLO_DTYPE_BF16 ? 2 : 4;
    YOLO_REQUIRE((((uintptr_t)x | (uintptr_t)weight | (uintptr_t)out | (uintptr_t)residual) & (z - 1)) == 0 &&
                     ((uintptr_t)bias & (bias_dtype == YOLO_DTYPE_BF16 ? 1 : 3)) == 0,
                 YOLO_ERR_ARG, "linear: a pointer is not aligned to its element");
    LinK k;
    k.x = (const char*)x; k.w = (const char*)weight; k.bias = bias; k.res = (const char*)residual; k.out = (char*)out;
    k.x_ld = x_ld * z; k.w_ld = weight_ld * z; k.res_ld = residual_ld * z; k.out_ld = out_ld * z;
    k.M = M; k.N = N; k.K = K;
    k.bias_bf16 = bias_dtype == YOLO_DTYPE_BF16; k.act = activation;
    k.vec_out = aligned16(out) && k.out_ld % 16 == 0 && (!residual || (aligned16(residual) && k.res_ld % 16 == 0));
    k.ntm = k.ntn = 0;
    const bool al = aligned16(x) && aligned16(weight) && k.x_ld % 16 == 0 && k.w_ld % 16 == 0 && (long long)K * z % 16 == 0;
    return dtype == YOLO_DTYPE_BF16 ? launch_linear<true>(k, al, (hipStream_t)stream) : launch_linear<false>(k, al, (hipStream_t)stream);
}
