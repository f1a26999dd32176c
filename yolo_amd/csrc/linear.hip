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
    unsigned ntm, ntn;
};

// gelu(v) = v * Phi(v) = v/2 * erfc(-v / sqrt 2).  f32 results take the library's erfcf (no cancellation in the negative tail).
// For bf16 results: max(v, 0) - |v| * e, e = erfc(|v| / sqrt 2) / 2 = t (a1 + t (a2 + ...)) exp(-v^2 / 2), t = 1 / (1 + 0.296 |v|), the six
// coefficients fitted here over 0 <= |v| <= 16 so that the error of e stays within 2^-21 and within 2^-14 of e itself: a tail of
// exponentially small results is as exact as the others, far inside the half step of bf16, 2^-8 of the value (evaluated in f32 over
// 200001 points: 3.2e-7 and 4.3e-5).  A form that bounds the absolute error alone is off by 1 % at -8.  One reciprocal, one
// exponential and twelve other instructions against about forty and a divergent branch: at 23104 x 4096 results the difference is a
// quarter of the whole product's time.  |v| is cut at 16, where the exponential is 0, so that +inf stays +inf and -inf gives 0.
template <bool BF16>
__device__ __forceinline__ float gelu(float v) {
    if constexpr (!BF16) {
        return v < -14.5f ? 0.f : 0.5f * v * erfcf(-0.70710678118654752f * v);      // 0 from there on, also at -inf
    } else {
        const float a = __builtin_fabsf(v);
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.296f, a, 1.0f));
        float p = __builtin_fmaf(-0.08246762f, t, 0.24361452f);
        p = __builtin_fmaf(p, t, -0.045269474f);
        p = __builtin_fmaf(p, t, 0.15600787f);
        p = __builtin_fmaf(p, t, 0.10943261f);
        p = __builtin_fmaf(p, t, 0.11868207f);
        const float e = p * t * __builtin_amdgcn_exp2f(v * v * -0.72134752f);      // log2(e) / 2
        return __builtin_fmaf(-__builtin_fminf(a, 16.0f), e, __builtin_fmaxf(v, 0.0f));
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

// A piece of an unaligned row: element k is at `at`.  The 16 bytes from element k on (global memory takes any address), or, where they
// would pass the row's end, the row's last 16 bytes; of a row of less than 16 bytes (SHORT) its elements, with zeros before them.
template <bool BF16, bool SHORT>
__device__ __forceinline__ u32x4 load_piece(const char* at, int k, int K) {
    typedef typename Elem<BF16>::type T;
    constexpr int P = Elem<BF16>::kPiece;
    const T* p = (const T*)at + min(0, K - P - k);
    if constexpr (SHORT) {
        typename std::conditional<BF16, bf16x8, f32x4>::type e = {};
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (j >= P - K) e[j] = p[j];
        return __builtin_bit_cast(u32x4, e);
    } else {
        u32x4 v;
        __builtin_memcpy(&v, p, 16);
        return v;
    }
}

// What load_piece read, as the piece of element k: moved down to its place, zeros past K.  One by one, the end's elements cost 2 us of 9 where
// the chain is short (1001 x 255 x 255).
template <bool BF16>
__device__ __forceinline__ u32x4 place_piece(u32x4 v, int k, int K) {
    constexpr int P = Elem<BF16>::kPiece, Z = 16 / P;
    const int excess = k + P - K;
    if (excess <= 0) return v;
    if (excess >= P) return u32x4{0, 0, 0, 0};
    const int bytes = excess * Z;                           // in 32-bit steps: see the masks of cross_attention_tile_kernel
    if (bytes & 8) v = u32x4{v[2], v[3], 0, 0};
    if (bytes & 4) v = u32x4{v[1], v[2], v[3], 0};
    if (bytes & 2) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    return v;
}

// ---- tiles of BM rows of x by BN rows of W through LDS ------------------------------------------------------------------------
// WR x WC waves, each (BM / WR) x (BN / WC); K in steps of 128 bytes, two LDS buffers, one barrier a step: the loads of the next
// step are issued before the products of this one.
// An LDS row is 128 bytes = 8 pieces, piece c of row r at slot c ^ (r & 7), so that the 16 rows a fragment read touches fall on
// all banks.  W is the MFMA's first operand: a lane then holds four consecutive outputs of one row of y.  The accumulators start
// from the bias.
// ALIGNED: rows of x and W start on 16 bytes and K is whole pieces; they go global -> LDS by DMA, pieces past K from a zero piece.
// Otherwise the pieces pass through registers.
//
// Measured, bf16: 8192^3 1.36 PFLOP/s with 256 x 256 tiles of 16 waves (64 x 64 each, 116 registers, one workgroup a CU), a fifth less with
// 128 x 128 (two a CU); the library's product reaches 1.65 on the same card.  23104 x 4096 x 1024 1.07 PFLOP/s, as the library, and with gelu
// 0.88: six rounds of 256 tiles, between which loads, stores and the activation are not covered by products.  173056 x 512 x 256 with gelu
// and residual 3.3 TB/s, bandwidth and the same gaps.  Persistent workgroups that fetch the next tile before the epilogue were slower (128
// registers do not hold both); f32 115 to 120 TFLOP/s at 23104 x 1024 x 512 (the library 100; 154 at 8192^3).
__device__ const u32x4 kZeroPiece = {0, 0, 0, 0};

// Swaps lane rows so that a lane that holds 4 outputs of each of two 16-wide tiles (a: tile i, b: tile i + 1, packed pairs) holds 8
// consecutive ones of one tile, and back: v_permlane16_swap is its own inverse.
__device__ __forceinline__ void swap_pairs(uint32_t& a, uint32_t& b) {
    const auto sw = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = sw[0];
    b = sw[1];
}

// workgroups of a CU by LDS, at most 4
constexpr int lin_blocks(int bm, int bn) { return bm + bn > 320 ? 1 : bm + bn > 160 ? 2 : 4; }

template <bool BF16, int BM, int BN, int WR, int WC, bool ALIGNED>
__global__ __launch_bounds__(WR* WC * 64, lin_blocks(BM, BN) * WR * WC / 4) void linear_tile_kernel(LinK p) {
    typedef typename Elem<BF16>::type T;
    constexpr int NT = WR * WC * 64, P = Elem<BF16>::kPiece, BK = 8 * P, RPI = NT / 8;
    constexpr int TM = BM / WR / 16, TN = BN / WC / 16, GM = 8;
    constexpr int LX = BM / RPI, LW = BN / RPI;             // pieces of x / W a thread stages per step
    constexpr int BUF = (BM + BN) * 128;
    static_assert(BM % RPI == 0 && BN % RPI == 0 && RPI % 8 == 0, "whole pieces per thread");
    static_assert(TN % 2 == 0, "bf16 stores pair two column tiles");
    extern __shared__ char lds[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // tiles in groups of GM row tiles by all column tiles, rows first: what an XCD runs at a time is a block about as high as wide,
    // which reads the fewest operand rows through its L2
    const unsigned tile = xcd_chunk(blockIdx.x, p.ntm * p.ntn), group = tile / (GM * p.ntn), in = tile - group * GM * p.ntn;
    const unsigned gm = min((unsigned)GM, p.ntm - group * GM), tn = in / gm, tm = group * GM + in - tn * gm;
    const long long m0 = (long long)tm * BM;
    const int n0 = (int)tn * BN;
    const int nsteps = (p.K + BK - 1) / BK;
    const int fr = lane & 15, fh = lane >> 4;
    const int wm0 = (wave / WC) * (BM / WR), wn0 = (wave % WC) * (BN / WC);

    // staging: this thread's piece of rows r0 + RPI i.  Rows past the last one read the last one again: their results are not stored
    const int r0 = tid >> 3, kc = ((tid & 7) ^ (r0 & 7)) * P;
    const int x_ld = (int)p.x_ld, w_ld = (int)p.w_ld;
    const char *const xb = p.x + m0 * p.x_ld, *const wb = p.w + n0 * p.w_ld;
    uint32_t off[LX + LW];
    {
        const int mlast = (int)min((long long)BM, p.M - m0) - 1, nlast = min(BN, p.N - n0) - 1;
#pragma unroll
        for (int i = 0; i < LX + LW; ++i)
            off[i] = (uint32_t)((i < LX ? min(r0 + RPI * i, mlast) * x_ld : min(r0 + RPI * (i - LX), nlast) * w_ld) + kc * (int)sizeof(T));
    }
    u32x4 stage[ALIGNED ? 1 : LX + LW];
    auto issue = [&](int s, int buf) {
        const char *xs = xb + s * 128, *ws = wb + s * 128;
        char* const dst = lds + buf * BUF + wave * 1024;
        if constexpr (ALIGNED) {
            if ((s + 1) * BK <= p.K) {
#pragma unroll
                for (int i = 0; i < LX + LW; ++i) dma16((i < LX ? xs : ws) + off[i], dst + i * NT * 16);
            } else {
#pragma unroll
                for (int i = 0; i < LX + LW; ++i)
                    dma16(s * BK + kc < p.K ? (const void*)((i < LX ? xs : ws) + off[i]) : (const void*)&kZeroPiece, dst + i * NT * 16);
            }
        } else {
            if ((s + 1) * BK <= p.K) {
#pragma unroll
                for (int i = 0; i < LX + LW; ++i) __builtin_memcpy(&stage[i], (i < LX ? xs : ws) + off[i], 16);
            } else if (p.K >= P) {
#pragma unroll
                for (int i = 0; i < LX + LW; ++i) stage[i] = load_piece<BF16, false>((i < LX ? xs : ws) + off[i], s * BK + kc, p.K);
            } else {
#pragma unroll
                for (int i = 0; i < LX + LW; ++i) stage[i] = load_piece<BF16, true>((i < LX ? xs : ws) + off[i], s * BK + kc, p.K);
            }
        }
    };
    auto settle = [&](int s, int buf) {                     // not ALIGNED: registers -> LDS
        if constexpr (!ALIGNED) {
            if ((s + 1) * BK > p.K) {
#pragma unroll
                for (int i = 0; i < LX + LW; ++i) stage[i] = place_piece<BF16>(stage[i], s * BK + kc, p.K);
            }
#pragma unroll
            for (int i = 0; i < LX + LW; ++i) *(u32x4*)(lds + buf * BUF + (i * NT + tid) * 16) = stage[i];
        }
    };
    f32x4 acc[TN][TM];
    issue(0, 0);
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        f32x4 bv = {0.f, 0.f, 0.f, 0.f};
        if (p.bias) {
#pragma unroll
            for (int r = 0; r < 4; ++r) bv[r] = load_param(p.bias, p.bias_bf16, min(n0 + wn0 + i * 16 + fh * 4 + r, p.N - 1));
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = bv;
    }
    settle(0, 0);
    for (int s = 0; s < nsteps; ++s) {
        const int buf = s & 1;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (s + 1 < nsteps) issue(s + 1, buf ^ 1);
        const char* bx = lds + buf * BUF;
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
        // schedule: all fragments of the first half step, then those of the second between its products
        constexpr int kReads = TM + TN, kProducts = TM * TN * (BF16 ? 1 : 4);
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);                     // LDS reads
#pragma unroll
        for (int q = 0; q < kReads; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x8, kProducts / kReads, 0);       // MFMAs
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 2 * kProducts - kProducts / kReads * kReads, 0);
        if (s + 1 < nsteps) settle(s + 1, buf ^ 1);
    }

    // epilogue in registers: lane holds y[m][n .. n+3] for m = wm0 + 16 j + fr, n = wn0 + 16 i + 4 fh.  Results leave and residuals come in
    // pieces of 16 bytes wherever their rows start (global memory takes any address).  bf16: after swap_pairs a lane's piece of the
    // tile pair i, i + 1 is 8 columns of one of the two; f32: 4 columns of each.
    char* const ob = p.out + m0 * p.out_ld + (long long)n0 * sizeof(T);
    const char* const rb = p.res + m0 * p.res_ld + (long long)n0 * sizeof(T);
    const int pc = wn0 + (BF16 ? (fh & 1) * 16 + (fh >> 1) * 8 : fh * 4);           // first column of this lane's piece of pair 0
    const uint32_t ro = (uint32_t)(wm0 + fr) * (uint32_t)p.res_ld + (uint32_t)pc * (uint32_t)sizeof(T);
    const uint32_t oo = (uint32_t)(wm0 + fr) * (uint32_t)p.out_ld + (uint32_t)pc * (uint32_t)sizeof(T);
    const int mleft = (int)min((long long)BM, p.M - m0) - wm0 - fr, nleft = min(BN, p.N - n0) - pc;    // rows / columns from this lane's first on
    auto finish = [&](auto inner) {
        auto whole = [&](int j, int i) { return inner.value || (j * 16 < mleft && i * 16 + P <= nleft); };
        // residual pieces come in two halves of the rows, the second requested before the first half's results are stored:
        // a load behind a store would wait for it
        constexpr int C = TM % 2 == 0 ? 2 : 1, CM = TM / C;
        u32x4 rv[CM][TN / 2], rw[BF16 ? 1 : CM][BF16 ? 1 : TN / 2];
        auto fetch_res = [&](int c) {
            if (!p.res) return;
#pragma unroll
            for (int j = 0; j < CM; ++j)
#pragma unroll
                for (int i = 0; i < TN; i += 2) {
                    const char* q = rb + (long long)(c * CM + j) * 16 * p.res_ld + i * 16 * (int)sizeof(T) + ro;
                    rv[j][i / 2] = u32x4{0, 0, 0, 0};
                    if (whole(c * CM + j, i)) __builtin_memcpy(&rv[j][i / 2], q, 16);
                    if constexpr (!BF16) {
                        rw[j][i / 2] = u32x4{0, 0, 0, 0};
                        if (whole(c * CM + j, i + 1)) __builtin_memcpy(&rw[j][i / 2], q + 64, 16);
                    }
                }
        };
        fetch_res(0);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            u32x4 ov[CM][TN / 2], ow[BF16 ? 1 : CM][BF16 ? 1 : TN / 2];
            with_act(p.act, [&](auto mode) {
                constexpr int ACT = decltype(mode)::value;
#pragma unroll
                for (int j = 0; j < CM; ++j)
#pragma unroll
                    for (int i = 0; i < TN; i += 2) {
                        f32x4 v0, v1;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            v0[r] = activate<BF16, ACT>(acc[i][c * CM + j][r]);
                            v1[r] = activate<BF16, ACT>(acc[i + 1][c * CM + j][r]);
                        }
                        if constexpr (BF16) {
                            if (p.res) {                // brought from store order to accumulator order, added before the one rounding
                                uint32_t q0 = rv[j][i / 2][0], q1 = rv[j][i / 2][1], q2 = rv[j][i / 2][2], q3 = rv[j][i / 2][3];
                                swap_pairs(q0, q2);
                                swap_pairs(q1, q3);
                                v0 += f32x4{bf16_lo(q0), bf16_hi(q0), bf16_lo(q1), bf16_hi(q1)};
                                v1 += f32x4{bf16_lo(q2), bf16_hi(q2), bf16_lo(q3), bf16_hi(q3)};
                            }
                            uint32_t a0 = pack_bf16(v0[0], v0[1]), a1 = pack_bf16(v0[2], v0[3]);
                            uint32_t b0 = pack_bf16(v1[0], v1[1]), b1 = pack_bf16(v1[2], v1[3]);
                            swap_pairs(a0, b0);
                            swap_pairs(a1, b1);
                            ov[j][i / 2] = u32x4{a0, a1, b0, b1};
                        } else {
                            if (p.res) {
                                v0 += __builtin_bit_cast(f32x4, rv[j][i / 2]);
                                v1 += __builtin_bit_cast(f32x4, rw[j][i / 2]);
                            }
                            ov[j][i / 2] = __builtin_bit_cast(u32x4, v0);
                            ow[j][i / 2] = __builtin_bit_cast(u32x4, v1);
                        }
                    }
            });
            if (c + 1 < C) fetch_res(c + 1);
#pragma unroll
            for (int j = 0; j < CM; ++j)
#pragma unroll
                for (int i = 0; i < TN; i += 2) {
                    char* o = ob + (long long)(c * CM + j) * 16 * p.out_ld + i * 16 * (int)sizeof(T) + oo;
                    if (whole(c * CM + j, i)) __builtin_memcpy(o, &ov[j][i / 2], 16);
                    if constexpr (!BF16) {
                        if (whole(c * CM + j, i + 1)) __builtin_memcpy(o + 64, &ow[j][i / 2], 16);
                    }
                }
        }
    };
    if (m0 + BM <= p.M && n0 + BN <= p.N) finish(std::true_type{});
    else finish(std::false_type{});
    // the last N % P columns, element by element: one 16-wide tile of one wave column
    const int tail = p.N / P * P;
    if (tail < p.N && tail >= n0 + wn0 && tail < n0 + wn0 + TN * 16) {
        with_act(p.act, [&](auto mode) {
            constexpr int ACT = decltype(mode)::value;
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const int n = n0 + wn0 + i * 16 + fh * 4;
                if ((tail - n0 - wn0) / 16 != i || n + 3 < tail) continue;
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    const long long m = m0 + wm0 + j * 16 + fr;
                    if (m >= p.M) continue;
                    T* o = (T*)(p.out + m * p.out_ld);
                    const T* q = (const T*)(p.res + m * p.res_ld);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (n + r < tail || n + r >= p.N) continue;
                        float v = activate<BF16, ACT>(acc[i][j][r]);
                        if (p.res) v += load_f32(q + n + r);
                        o[n + r] = (T)v;
                    }
                }
            }
        });
    }
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
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned tile = xcd_chunk(blockIdx.x, p.ntm * p.ntn);
    const unsigned tm = tile % p.ntm, tn = tile / p.ntm;     // row tiles of one W tile next to each other
    const long long m0 = (long long)tm * BM;
    const int n0 = (int)tn * BN;
    const int fr = lane & 15, fh = lane >> 4;
    const int nslices = (p.K + BK - 1) / BK;
    // rows past the last one read the last one again: their results are not stored
    const char* xr[TM];
    const char* wr[TN];
#pragma unroll
    for (int j = 0; j < TM; ++j) xr[j] = p.x + min(m0 + j * 16 + fr, p.M - 1) * p.x_ld;
#pragma unroll
    for (int i = 0; i < TN; ++i) wr[i] = p.w + (long long)min(n0 + i * 16 + fr, p.N - 1) * p.w_ld;
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;                                     // slices in flight; those past K are zeros
    auto walk = [&](auto is_short) {
        auto piece = [&](const char* row, int k) {
            if constexpr (ALIGNED) return *(k < p.K ? (const u32x4*)(row + (long long)k * sizeof(T)) : &kZeroPiece);
            else return load_piece<BF16, decltype(is_short)::value>(row + (long long)k * sizeof(T), k, p.K);
        };
        for (int s = wave; s < nslices; s += U * W) {
            u32x4 fx[U][TM], fw[U][TN];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (s + u * W) * BK + fh * P;
                if (!ALIGNED && s + u * W >= nslices) break;
#pragma unroll
                for (int i = 0; i < TN; ++i) fw[u][i] = piece(wr[i], k);
#pragma unroll
                for (int j = 0; j < TM; ++j) fx[u][j] = piece(xr[j], k);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k0 = (s + u * W) * BK;
                if constexpr (!ALIGNED) {
                    if (s + u * W >= nslices) break;
                    if (k0 + BK > p.K) {
#pragma unroll
                        for (int i = 0; i < TN; ++i) fw[u][i] = place_piece<BF16>(fw[u][i], k0 + fh * P, p.K);
#pragma unroll
                        for (int j = 0; j < TM; ++j) fx[u][j] = place_piece<BF16>(fx[u][j], k0 + fh * P, p.K);
                    }
                }
#pragma unroll
                for (int i = 0; i < TN; ++i)
#pragma unroll
                    for (int j = 0; j < TM; ++j) acc[i][j] = mma<BF16>(fw[u][i], fx[u][j], acc[i][j]);
            }
        }
    };
    if (ALIGNED || p.K >= P) walk(std::false_type{});
    else walk(std::true_type{});
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
    YOLO_REQUIRE(launchable(ntm * ntn, WR * WC * 64), YOLO_ERR_UNSUPPORTED, "linear: %llu tiles are more than one launch takes", ntm * ntn);
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
    YOLO_REQUIRE(launchable(ntm * ntn, 512), YOLO_ERR_UNSUPPORTED, "linear: %llu tiles are more than one launch takes", ntm * ntn);
    k.ntm = (unsigned)ntm;
    k.ntn = (unsigned)ntn;
    hipLaunchKernelGGL((linear_direct_kernel<BF16, TM, TN, ALIGNED>), dim3(k.ntm * k.ntn), dim3(512), 0, stream, k);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}

// Tile by the time that the rounds of its tiles on the 256 CUs take.
// bf16, in units of a 128 x 128 tile's share of a CU: one 256 x 256 tile a CU takes 4 (1.3 PFLOP/s at 8192^3, 128 x 128 1.1 with twice the
// operand traffic), two of 192 x 128 3.35, two of 128 x 128 2.55, four of 64 x 64 1.75: fitted to 67 shapes (600 to 200000 rows, 48 to 8192
// wide), where the choice is 2 % from the best of six tiles on average.  Measured (us for 256 / 192 / 128 / 64): 23104 x 4096 x 1024 217 / 227 /
// 244 / 319, 5000 x 2048 x 2048 55 / 45 / 58 / 69, 8000 x 1024 x 1024 30 / 26 / 23 / 34, 2704 x 1024 x 256 15.5 / 9.4 / 8.8 / 6.9.
// f32 is bound by its products: rounds of one tile a CU times the tile, 96 x 64 counted 2 % and 128 x 128 4 % cheaper for their fewer operand reads.
// Measured (us for 128 / 96 / 64): 23104 x 1024 x 512 207 / 210 / 212, 5408 x 512 x 512 39 / 32 / 35, 1500 x 1024 x 1024 69 / 32 / 40,
// 2194 x 864 x 1680 114 / 89 / 64; within 1.2 % of the best of six tiles on average over 44 of the shapes.
// Few outputs go to the direct kernel, which splits K inside a workgroup: up to 512 tiles of 16 x 16 (40 x 1024 x 1024: 4.1 against 6.7 in
// 32 x 32 and 8.2 in 64 x 64), up to 256 of 32 x 32 (300 x 512 x 1024: 7.4 against 11.2; 700 x 512 x 512, 352 tiles: 9.0 against 7.9), 512 in f32, whose products
// take four times as long (300 x 512 x 1024: 10.8 against 24.6).
// Up to 32 columns take tiles of 64 x 32, as a wider one multiplies rows of W that are not there: 57289 x 32 x 1008 in f32 55 us (4.3 TB/s)
// against 83 with 64 x 64, in bf16 31 against 34; 100000 x 32 x 64 in bf16 7.3 against 8.2.
// The direct kernel forms 64-bit addresses; the tile kernel offsets rows of a tile in 32 bits and takes strides up to 4 MB.
template <bool BF16>
static int launch_linear(const LinK& k, bool aligned, hipStream_t stream) {
    auto tiles = [&](int e) { return (unsigned long long)((k.M + e - 1) / e) * ((k.N + e - 1) / e); };
    const long long kMaxStride = 1ll << 22;
    const bool wide = k.x_ld > kMaxStride || k.w_ld > kMaxStride || k.out_ld > kMaxStride || (k.res && k.res_ld > kMaxStride);
    if (tiles(16) <= 512) return aligned ? launch_direct<BF16, 1, 1, true>(k, stream) : launch_direct<BF16, 1, 1, false>(k, stream);
    if (tiles(32) <= (BF16 ? 256 : 512) || wide) return aligned ? launch_direct<BF16, 2, 2, true>(k, stream) : launch_direct<BF16, 2, 2, false>(k, stream);
    if (k.N <= 32) return aligned ? launch_tile<BF16, 64, 32, 4, 1, true>(k, stream) : launch_tile<BF16, 64, 32, 4, 1, false>(k, stream);
    auto rounds = [&](int bm, int bn, int slots) {
        const unsigned long long n = (unsigned long long)((k.M + bm - 1) / bm) * ((k.N + bn - 1) / bn);
        return (double)((n + slots - 1) / slots);
    };
    // where pieces pass through registers (operands out of HBM), sixteen waves of 32 x 32 take 100 us against 103 with four of 64 x 64 at 23104 x 1024 x 1023, and
    // eight of 16 x 32 7.1 against 8.1 with four of 32 x 32 at 1001 x 255 x 255; in f32 likewise 207 against 215 at 23104 x 1024 x 512 and 35 against 37
    // at 5408 x 512 x 512
    if constexpr (BF16) {
        const double c256 = rounds(256, 256, 256) * 4.0, c192 = rounds(192, 128, 512) * 3.35, c128 = rounds(128, 128, 512) * 2.55;
        const double c64 = rounds(64, 64, 1024) * 1.75;
        if (!aligned) return c128 <= c64 ? launch_tile<BF16, 128, 128, 4, 4, false>(k, stream) : launch_tile<BF16, 64, 64, 4, 2, false>(k, stream);
        if (c256 <= c192 && c256 <= c128 && c256 <= c64) return launch_tile<BF16, 256, 256, 4, 4, true>(k, stream);
        if (c192 <= c128 && c192 <= c64) return launch_tile<BF16, 192, 128, 4, 2, true>(k, stream);
        return c128 <= c64 ? launch_tile<BF16, 128, 128, 2, 2, true>(k, stream) : launch_tile<BF16, 64, 64, 2, 2, true>(k, stream);
    } else {
        const double c128 = rounds(128, 128, 256) * 4.0 * 0.96, c96 = rounds(96, 64, 256) * 1.5 * 0.98, c64 = rounds(64, 64, 256);
        if (!aligned) return c128 <= c64 ? launch_tile<BF16, 128, 128, 4, 4, false>(k, stream) : launch_tile<BF16, 64, 64, 4, 2, false>(k, stream);
        if (c128 <= c96 && c128 <= c64) return launch_tile<BF16, 128, 128, 4, 4, true>(k, stream);
        return c96 <= c64 ? launch_tile<BF16, 96, 64, 2, 2, true>(k, stream) : launch_tile<BF16, 64, 64, 4, 2, true>(k, stream);
    }
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
    k.ntm = k.ntn = 0;
    const bool al = aligned16(x) && aligned16(weight) && k.x_ld % 16 == 0 && k.w_ld % 16 == 0 && (long long)K * z % 16 == 0;
    return dtype == YOLO_DTYPE_BF16 ? launch_linear<true>(k, al, (hipStream_t)stream) : launch_linear<false>(k, al, (hipStream_t)stream);
}
