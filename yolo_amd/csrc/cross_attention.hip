// yolo_cross_attention: o = softmax(scale * q k^T) v over the kept keys of another sequence, query heads in groups that share a
// key / value head.
//
// Mathematics: one pass over the keys with the running maximum m and sum l of the softmax: with m' = max(m, max s),
// o <- o exp(m - m') + sum exp(s - m') v and l likewise, result o / l.  Scores, m, l and o are f32.  A key is kept when its
// index is below key_lens[b] and its key_mask byte is set; what is not kept is never multiplied (its score is replaced, its
// value row not used), so that infinities and NaN there stay out.  A row without a kept key is zero.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "layer_common.h"

namespace yolo {

struct AttnK {
    const char* q;
    const char* k;
    const char* v;
    char* out;                          // [B, Lq, Hq, D] packed
    const int32_t* lens;                // [B] or nullptr
    const uint8_t* mask;                // [B, Lk] or nullptr
    long long qb, ql, qh, kb, kl, kh, vb, vl, vh;   // element strides
    int B, Lq, Lk, Hq, Hk, D, G;        // G = Hq / Hk
    float scale;
    // matrix-core kernels
    uint32_t q_and, q_xor;              // applied to every 32 bits of q: a negative or zero scale is folded into q
    float scale2;                       // |scale| * log2(e) (log2(e) for scale 0): weights are 2^(scale2 * (s - max))
    int rtiles, splits, tps;            // row tiles per (image, key head), key splits, key tiles per split
    float* part;                        // [splits][B*Lq*Hq][D] unnormalised results
    float2* ml;                         // [splits][B*Lq*Hq] (maximum, sum); sum -1: no kept key in the split
};

// keys of image b that can be kept: [0, n)
__device__ __forceinline__ int key_count(const AttnK& p, int b) {
    int n = p.Lk;
    if (p.lens) n = max(0, min(n, p.lens[b]));
    return n;
}

// Any D <= 256, any alignment: one wave per (image, query, head).  Lane = key for the scores, lane + 64 i = element of the
// head for the products with v; only kept keys are read.
template <bool BF16>
__global__ __launch_bounds__(256) void cross_attention_general_kernel(AttnK p) {
    typedef typename Elem<BF16>::type T;
    __shared__ float qs[4][256];
    __shared__ float ps[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * 4 + wave;
    const long long rows = (long long)p.B * p.Lq * p.Hq;
    const bool in = row < rows;
    const int h = in ? (int)(row % p.Hq) : 0, hk = h / p.G;
    const long long bl = in ? row / p.Hq : 0;
    const int l = (int)(bl % p.Lq), b = (int)(bl / p.Lq);
    const T* q = (const T*)p.q + b * p.qb + l * p.ql + h * p.qh;
    for (int d = lane; d < p.D; d += 64) qs[wave][d] = load_f32(q + d) * p.scale;
    __syncthreads();
    if (!in) return;                    // no workgroup barrier below
    const T* kp = (const T*)p.k + b * p.kb + hk * p.kh;
    const T* vp = (const T*)p.v + b * p.vb + hk * p.vh;
    const int n = key_count(p, b);
    float m = -__builtin_inff(), sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    bool any = false;
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane;
        const bool keep = j < n && (!p.mask || p.mask[(long long)b * p.Lk + j]);
        unsigned long long kept = __ballot(keep);
        if (!kept) continue;
        any = true;
        float s = -__builtin_inff();
        if (keep) {
            const T* kr = kp + (long long)j * p.kl;
            s = 0.f;
            for (int d = 0; d < p.D; ++d) s = __builtin_fmaf(qs[wave][d], load_f32(kr + d), s);
        }
        float mt = s;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) mt = fmaxf(mt, __shfl_xor(mt, x));
        const float mn = fmaxf(m, mt), base = mn == -__builtin_inff() ? 0.f : mn;
        const float e = expf(s - base), c = expf(m - base);
        float st = keep ? e : 0.f;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) st += __shfl_xor(st, x);
        sum = sum * c + st;
        m = mn;
        ps[wave][lane] = e;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= c;
        while (kept) {
            const int jj = __builtin_ctzll(kept);
            kept &= kept - 1;
            const float pj = ps[wave][jj];
            const T* vr = vp + (long long)(j0 + jj) * p.vl;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = lane + 64 * i;
                if (d < p.D) o[i] = __builtin_fmaf(pj, load_f32(vr + d), o[i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    T* out = (T*)p.out + row * p.D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < p.D) out[d] = (T)(any ? o[i] / sum : 0.f);
    }
}

// ---- tiles on the matrix cores --------------------------------------------------------------------------------------------------
// A workgroup of WAVES waves takes 32 WAVES query rows of one (image, key head) - row r is query r / G, head r % G of the group,
// so that the heads that share k and v share their tiles - and walks KT keys at a time; k and v tiles are double-buffered in
// LDS by DMA, one barrier per tile.
//
// Scores are computed transposed, S^T = K Q^T on 32x32 MFMAs: lane l then holds 16 scores of ONE query (l % 32) per 32 keys (keys
// 8 b + 4 (l / 32) + i at register 4 b + i), so maximum and sum are in-lane but for one exchange with lane l ^ 32, and the
// rescaling factor of o is a lane's own scalar.  P^T in that layout IS the second operand of O^T = V^T P^T if the reduction
// index runs over the keys in the order the lane holds them; v is read to match: bf16 by ds_read_b64_tr_b16 (4 keys x 16
// elements transposed per 16 lanes), f32 by single words.
//
// The running maximum is only raised when a score exceeds it by 2^8 in weight: weights stay below 2^8, which costs no precision
// (they are floating point) and most tiles skip the rescaling of o.
// bf16: the weights are rounded to bf16 for the second product, at most 2^-8 of each and of either sign, which is the size of the
// rounding of the result; their sum is taken of the f32 values.  The error of a result against float64 is 0.0023 of its size with that, 0.0017
// without.  Where a head group has no more than 32 rows (WHOLE) the weights go in as two bf16, the upper 16 bits and the rest, within 2^-15
// of themselves, and both are multiplied: such calls wait for k and v (one query of 16 / 4 heads of 64 over 3549 keys 10.0 against 9.4 us,
// 64 of them 50.0 against 49.8).  With more rows the products bound the call and a third half as much again shows: 8 x 676 over 2704 keys, 8 heads
// of 64, 77 against 58 us, 8 x 2704 over 5776 of 128 718 against 548.
//
// CS > 1: the columns of v and of the result are divided over CS workgroups, each of which forms all the scores.  At D = 256 that halves
// the registers of o: two workgroups of a CU instead of one hide each other's latencies in bf16, 4 x 1000 x 2000 keys of 4 heads 70 us
// against 83, 8 x 1444 x 2704 of 8 heads 420 against 460.  f32 takes it where the tiles do not fill the GPU (4 x 559 x 30 keys of 2 heads 16.8 us
// against 23.2), not elsewhere (8 x 1444 x 1444 of 4 heads 1093 against 906: its products bound it).
//
// LDS rows are the next power of two of the head size.  k: 16-byte piece c of a row at c ^ f(row) so that 16 rows' pieces fall on
// all banks; v: 64-byte (f32: 128-byte) blocks exchanged likewise for the transposed reads of four rows at a time.
__device__ const u32x4 kZeroPiece = {0, 0, 0, 0};

template <bool BF16, int DC> struct AttnTile {
    static constexpr int Z = BF16 ? 2 : 4, P = 16 / Z;                              // bytes and elements of a piece
    static constexpr int ROW = DC * Z <= 64 ? 64 : DC * Z <= 128 ? 128 : DC * Z <= 256 ? 256 : DC * Z <= 512 ? 512 : 1024;
    static constexpr int PCS = ROW / 16, KT = ROW >= 512 ? 32 : 64;                  // pieces of an LDS row, keys per tile
    static constexpr int RPL = ROW >= 256 ? 1 : 256 / ROW;                          // rows per 256 bytes (all banks)
    static constexpr int TILE = KT * ROW;                                           // bytes of one k or v tile
    static constexpr int BLK = BF16 ? 4 : 8;                                        // pieces of a v block
    static __device__ __forceinline__ int kpiece(int row, int c) { return c ^ ((row / RPL) & (PCS - 1)); }
    static __device__ __forceinline__ int vpiece(int row, int c) {
        constexpr int NB = PCS / BLK;                                               // blocks of a row
        if constexpr (NB <= 1) return c;
        else if constexpr (BF16) return c ^ ((((row & 3) / RPL) & (NB - 1)) * BLK);
        else return c ^ (((row >> 2) & 1) * BLK);
    }
};

template <bool BF16, int DC, int WAVES, int MW, int CS, bool WHOLE>
__global__ __launch_bounds__(WAVES * 64, MW) void cross_attention_tile_kernel(AttnK p) {
    typedef typename Elem<BF16>::type T;
    typedef AttnTile<BF16, DC> L;                           // k
    typedef AttnTile<BF16, DC / CS> LV;                     // v: DC / CS columns of as many keys
    constexpr int P = L::P, PCS = L::PCS, KT = L::KT, NT = WAVES * 64;
    constexpr int QS = DC / (2 * P);                        // k steps of S: two pieces (one per lane half) each
    constexpr int DT = DC / CS / 32, KB = KT / 32;          // 32-wide tiles of o, 32-key tiles of S
    constexpr int RPI = NT / PCS;                           // rows a pass of all threads stages
    constexpr int NI = KT / RPI, VRPI = NT / LV::PCS, VNI = KT / VRPI, VTILE = KT * LV::ROW;
    static_assert(KT % RPI == 0 && KT % VRPI == 0, "whole passes");
    extern __shared__ char lds[];                           // k0 k1 v0 v1

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    unsigned id = xcd_chunk(blockIdx.x, gridDim.x);
    const int c0 = (int)(id % CS) * (DC / CS);              // first column of v and of the result
    id /= CS;
    const int rt = (int)(id % p.rtiles);
    id /= p.rtiles;
    const int split = (int)(id % p.splits);
    id /= p.splits;
    const int hk = (int)(id % p.Hk), b = (int)(id / p.Hk);
    const int rows = p.Lq * p.G;
    const int n = key_count(p, b);
    const int t0 = split * p.tps;
    const int t1 = min((n + KT - 1) / KT, t0 + p.tps);

    // query rows of this wave -> registers (operand layout: column = row of q, 16-byte piece 2 step + half)
    const int row = rt * (32 * WAVES) + wave * 32 + col;
    long long orow;                                         // row of the packed output
    u32x4 fq[QS];
    {
        const int r = min(row, rows - 1), l = r / p.G, h = hk * p.G + r % p.G;
        orow = ((long long)b * p.Lq + l) * p.Hq + h;
        const char* q = p.q + (b * p.qb + l * p.ql + h * p.qh) * (long long)sizeof(T);
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            const int c = 2 * s + half;
            u32x4 v = *(c * P < p.D ? (const u32x4*)(q + c * 16) : &kZeroPiece);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (v[j] & p.q_and) ^ p.q_xor;
            fq[s] = v;
        }
    }

    f32x16 o[DT];
    float mref = -__builtin_inff(), sum = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;

    // staging: thread covers slot tid % PCS of rows tid / PCS + RPI i; of v likewise
    const int r0 = tid / PCS, slot = tid % PCS, vr0 = tid / LV::PCS, vslot = tid % LV::PCS;
    const long long kls = p.kl * (long long)sizeof(T), vls = p.vl * (long long)sizeof(T);
    const char* kbase = p.k + (b * p.kb + hk * p.kh) * (long long)sizeof(T);
    const char* vbase = p.v + (b * p.vb + hk * p.vh + c0) * (long long)sizeof(T);
    const uint8_t* mrow = p.mask ? p.mask + (long long)b * p.Lk : nullptr;
    auto mask_byte = [&](int t) {                           // lane = key of tile t; 0 beyond the last key
        const int j = t * KT + lane;
        return (mrow && lane < KT && j < n) ? (int)mrow[j] : 0;
    };
    // The mask of a tile is the wave's, in scalar registers, and is read in 32-bit words: a 64-bit shift by a vector count gave wrong masks
    // where the count sat in the last of 256 registers and two such waves filled a SIMD's register file.
    auto kept_bits = [&](int t, int mb) -> unsigned long long {
        unsigned long long bits;
        if (mrow) {
            bits = __ballot(mb != 0);
        } else {
            const int left = __builtin_amdgcn_readfirstlane(n - t * KT);
            bits = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1ull;
        }
        return (unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(bits >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)bits);
    };
    auto kept_row = [](unsigned long long bits, int r) {
        const uint32_t word = KT == 64 && r >= 32 ? (uint32_t)(bits >> 32) : (uint32_t)bits;
        return ((word >> (r & 31)) & 1u) != 0;
    };
    const unsigned long long full = KT == 64 ? ~0ull : 0xffffffffull;
    const bool padded = p.D * L::Z != L::ROW;
    auto issue = [&](int t, int buf, unsigned long long kept) {
        char* kd = lds + buf * L::TILE + wave * 1024;
        char* vd = lds + 2 * L::TILE + buf * VTILE + wave * 1024;
        const char* ks = kbase + ((long long)t * KT + r0) * kls;
        const char* vs = vbase + ((long long)t * KT + vr0) * vls;
        auto each_piece = [&](auto plain) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = r0 + i * RPI, c = L::kpiece(r, slot);
                const char* g = ks + (long long)(i * RPI) * kls + c * 16;
                if constexpr (!plain.value) g = kept_row(kept, r) && c * P < p.D ? g : (const char*)&kZeroPiece;
                dma16(g, kd + i * NT * 16);
            }
#pragma unroll
            for (int i = 0; i < VNI; ++i) {
                const int r = vr0 + i * VRPI, c = LV::vpiece(r, vslot);
                const char* g = vs + (long long)(i * VRPI) * vls + c * 16;
                if constexpr (!plain.value) g = kept_row(kept, r) && c0 + c * P < p.D ? g : (const char*)&kZeroPiece;
                dma16(g, vd + i * NT * 16);
            }
        };
        if (!padded && (kept & full) == full) each_piece(std::true_type{});
        else each_piece(std::false_type{});
    };

    bool any = false;
    unsigned long long kept = 0;
    int mb = 0;
    if (t0 < t1) {
        kept = kept_bits(t0, mask_byte(t0));
        issue(t0, 0, kept);
        mb = mask_byte(t0 + 1);
    }
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        const unsigned long long next = kept_bits(t + 1, mb);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (t + 1 < t1) {
            issue(t + 1, buf ^ 1, next);
            mb = mask_byte(t + 2);
        }
        const char* kt = lds + buf * L::TILE;
        const char* vt = lds + 2 * L::TILE + buf * VTILE;

        f32x16 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
            const int key = kb * 32 + col;
#pragma unroll
            for (int st = 0; st < QS; ++st) {
                const u32x4 fk = *(const u32x4*)(kt + key * L::ROW + L::kpiece(key, 2 * st + half) * 16);
                if constexpr (BF16) {
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fk), __builtin_bit_cast(bf16x8, fq[st]), s[kb], 0, 0, 0);
                } else {
                    const f32x4 a = __builtin_bit_cast(f32x4, fk), q = __builtin_bit_cast(f32x4, fq[st]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], q[j], s[kb], 0, 0, 0);
                }
            }
        }
        if ((kept & full) != full) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const uint32_t lane_keys = (uint32_t)(kept >> (32 * kb)) >> (4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kb][r] = lane_keys & (1u << (8 * (r >> 2) + (r & 3))) ? s[kb][r] : -__builtin_inff();
            }
        }
        any |= kept != 0;
        kept = next;

        float mt = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[kb][r]);
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const bool raise = (mt - mref) * p.scale2 > 8.f;    // false while both are -inf
        if (__any(raise)) {
            const float mn = fmaxf(mref, mt);
            const float c = mref == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((mref - mn) * p.scale2);
            mref = mn;
            sum *= c;
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= c;
        }
        // the rounding of `base` is a factor common to the row's weights, 2^(2^-24 base): past 4096 the maximum is subtracted first, as the
        // factor would overflow from 2^31 on
        float base = mref == -__builtin_inff() ? 0.f : mref * p.scale2;
        if (__any(fabsf(base) > 4096.f)) {
            const float mx = base == 0.f ? 0.f : mref;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kb][r] -= mx;
            base = 0.f;
        }
        float st = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], p.scale2, -base));
                s[kb][r] = e;
                st += e;
            }
        sum += st;

#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            if constexpr (BF16) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {               // 16 keys: registers 8 g .. 8 g + 7
                    u32x4 pk, rest;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float w0 = s[kb][8 * g + 2 * j], w1 = s[kb][8 * g + 2 * j + 1];
                        if constexpr (WHOLE) {
                            const uint32_t b0 = __float_as_uint(w0), b1 = __float_as_uint(w1);
                            pk[j] = b0 >> 16 | (b1 & 0xffff0000u);
                            rest[j] = pack_bf16(w0 - __uint_as_float(b0 & 0xffff0000u), w1 - __uint_as_float(b1 & 0xffff0000u));
                        } else {
                            pk[j] = pack_bf16(w0, w1);
                        }
                    }
                    const bf16x8 fp = __builtin_bit_cast(bf16x8, pk);
                    // lane's address for the transposed read: key row (lane / 4) % 4 of its four keys, 4 elements at 4 (lane % 4)
                    const int key = kb * 32 + 16 * g + 4 * half + ((lane >> 2) & 3);
#pragma unroll
                    for (int i = 0; i < DT; ++i) {
                        const int e = i * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;             // first element
                        const int c = e / 8, w = (e & 7) * 2;
                        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                            (__attribute__((address_space(3))) char*)vt + key * LV::ROW + LV::vpiece(key, c) * 16 + w));
                        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                            (__attribute__((address_space(3))) char*)vt + (key + 8) * LV::ROW + LV::vpiece(key + 8, c) * 16 + w));
                        typedef short s16x8 __attribute__((ext_vector_type(8)));
                        const bf16x8 fv = __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fv, fp, o[i], 0, 0, 0);
                        if constexpr (WHOLE) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fv, __builtin_bit_cast(bf16x8, rest), o[i], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = kb * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
                    for (int i = 0; i < DT; ++i) {
                        const int e = i * 32 + col;
                        const float fv = *(const float*)(vt + key * LV::ROW + LV::vpiece(key, e / 4) * 16 + (e & 3) * 4);
                        o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(fv, s[kb][r], o[i], 0, 0, 0);
                    }
                }
            }
        }
    }

    const long long total = (long long)p.B * p.Lq * p.Hq;
    const float l = sum + __shfl_xor(sum, 32);
    const bool in = row < rows;
    const bool parts = p.part != nullptr;
    const float f = parts ? 1.0f : any ? 1.0f / l : 0.f;
    if (in && parts && half == 0 && c0 == 0) p.ml[split * total + orow] = make_float2(mref, any ? l : -1.0f);
#pragma unroll
    for (int i = 0; i < DT; ++i) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            // registers 8 g + 0..3 and 8 g + 4..7 are elements 16 g + 4 half + 0..3 and + 8: after the exchange of lane halves a lane
            // holds 8 consecutive elements, 16 g + 8 half ..
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = o[i][8 * g + j] * f, c = o[i][8 * g + 4 + j] * f;
                const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(c), false, false);
                v[j] = __uint_as_float(sw[0]);
                v[4 + j] = __uint_as_float(sw[1]);
            }
            const int d = c0 + i * 32 + 16 * g + 8 * half;
            if (!in || d >= p.D) continue;              // D is whole groups of 8
            if (parts || !BF16) {
                float* dst = parts ? p.part + (split * total + orow) * p.D + d : (float*)p.out + orow * p.D + d;
                *(f32x4*)dst = f32x4{v[0], v[1], v[2], v[3]};
                *(f32x4*)(dst + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                u32x4 pk;
#pragma unroll
                for (int j = 0; j < 4; ++j) pk[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                *(u32x4*)((__bf16*)p.out + orow * p.D + d) = pk;
            }
        }
    }
}

// Joins the key splits of a row: a workgroup of WPR waves per row, lane = split for the maxima and sums, lane + 64 i = element for the
// results; a wave adds every WPR-th split with four loads in flight, the waves' sums are added in order: the result does not depend on
// the launch.
constexpr int kMaxSplits = 64, WPR = 4;

template <bool BF16>
__global__ __launch_bounds__(256) void cross_attention_join_kernel(AttnK p) {
    typedef typename Elem<BF16>::type T;
    __shared__ float sums[WPR][256];
    const int lane = threadIdx.x & 63, w0 = threadIdx.x >> 6;
    const long long total = (long long)p.B * p.Lq * p.Hq, row = blockIdx.x;
    const bool have = lane < p.splits;
    const float2 ml = have ? p.ml[lane * total + row] : make_float2(-__builtin_inff(), -1.0f);
    const bool kept = have && ml.y != -1.0f;                // a NaN sum is kept
    const bool any = __ballot(kept) != 0;
    float m = kept ? ml.x : -__builtin_inff();
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    // a split without a kept key has results 0; one whose kept scores are all -inf has maximum -inf, sum 0 and results 0, or a NaN sum
    const float w = !kept ? 0.f : ml.x != -__builtin_inff() ? __builtin_amdgcn_exp2f((ml.x - m) * p.scale2) : ml.y == 0.f ? 0.f : 1.f;
    float l = kept ? w * ml.y : 0.f;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = w0; s0 < p.splits; s0 += 4 * WPR) {
        float v[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int s = s0 + u * WPR, d = lane + 64 * i;
                v[u][i] = s < p.splits && d < p.D ? p.part[(s * total + row) * p.D + d] : 0.f;
            }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float ws = __shfl(w, (s0 + u * WPR) & 63);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(ws, v[u][i], o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[w0][lane + 64 * i] = o[i];
    __syncthreads();
    if (w0) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 1; x < WPR; ++x) o[i] += sums[x][lane + 64 * i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < p.D) ((T*)p.out)[row * p.D + d] = (T)(any ? o[i] / l : 0.f);
    }
}

// The same for up to 8 splits and many rows: a thread per four elements, all its loads in flight.
template <bool BF16>
__global__ __launch_bounds__(256) void cross_attention_join_rows_kernel(AttnK p) {
    typedef typename Elem<BF16>::type T;
    const long long total = (long long)p.B * p.Lq * p.Hq;
    const int quads = p.D / 4;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x, row = id / quads;
    const int d = (int)(id - row * quads) * 4;
    if (row >= total) return;
    float2 ml[8];
    f32x4 v[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        ml[s] = s < p.splits ? p.ml[s * total + row] : make_float2(-__builtin_inff(), -1.0f);
        v[s] = s < p.splits ? *(const f32x4*)(p.part + (s * total + row) * p.D + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float m = -__builtin_inff(), l = 0.f;
    bool any = false;
#pragma unroll
    for (int s = 0; s < 8; ++s)
        if (ml[s].y != -1.0f) {
            m = fmaxf(m, ml[s].x);
            any = true;
        }
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        if (ml[s].y == -1.0f) continue;
        const float w = ml[s].x != -__builtin_inff() ? __builtin_amdgcn_exp2f((ml[s].x - m) * p.scale2) : ml[s].y == 0.f ? 0.f : 1.f;
        l += w * ml[s].y;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(w, v[s][j], o[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = any ? o[j] / l : 0.f;
    T* out = (T*)p.out + row * p.D + d;
    if constexpr (BF16) *(u32x2*)out = u32x2{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
    else *(f32x4*)out = o;
}

// ---- plan: the tile shape and the number of key splits, by sizes and type alone ---------------------------------------------------
struct AttnPlan {
    int dc, waves, kt, rtiles, cs, splits, tps;     // cs: column parts of v
    bool few;                                       // no more than 32 rows of a head group
    size_t bytes;
};

// The number of key splits S is the one of least modelled time, in microseconds: rounds of workgroups times the tiles of one, and for
// S > 1 the join's launch and the traffic of the partial results.  Measured (bf16, us at S = 1 / 2 / 4): 32 x 100 queries of 8 heads of 64 over
// 3549 keys 76 / 60 / 68, 16 x 100 of 128 over 3549 100 / 67 / 63, 64 x 2704 of 64 over 80 keys 126 / 437 / 437; one query of 16
// heads of 64, 4 key heads: 9.1 at S = 1, 8.5 at 5 over 300 keys; 28 at 1, 8.9 at 12 over 1444; 64 at 1, 10 at 28 over 3549.
// Eight waves share a tile's loads where their larger row tiles still fill the CUs as well (8 x 2704 queries of 8 heads of 128: 524
// against 553), not over few tiles (80 keys, above: 153).
// Up to 32 rows of a head group (measured with weights of one bf16, which take 0.6 to 0.8 us less) need one wave, but four load a tile faster while CUs are free (one query of 16 / 4 heads of 64 over 3549 keys
// 9.4 against 10.3 us, 2 of 2 heads of 96 over 217: 8.4 against 13.2), and at 96 and more in bf16 as many workgroups of four waves fit a CU as of one;
// one-wave workgroups where they fill the CUs several times (16 x that query 19 against 23, f32 54 against 72).
static AttnPlan attn_plan(int dtype, int B, int Lq, int Lk, int Hq, int Hk, int D) {
    AttnPlan a;
    const bool bf16 = dtype == YOLO_DTYPE_BF16;
    a.dc = D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256;
    a.kt = a.dc * (bf16 ? 2 : 4) > 256 ? 32 : 64;
    const long long rows = (long long)Lq * (Hq / Hk), groups = (long long)B * Hk;
    auto rtiles = [&](int waves) { return (rows + 32 * waves - 1) / (32 * waves); };
    auto rounds = [](long long blocks, long long slots) { return (blocks + slots - 1) / slots; };
    const bool few = a.few = rows <= 32;
    const int tiles = (Lk + a.kt - 1) / a.kt;
    int wide = 4;                                           // waves of a workgroup where there are rows for more than one
    if (bf16 && a.dc >= 64 && a.dc <= 128 && tiles >= 8 && rtiles(8) * groups >= 512 && rounds(rtiles(8) * groups, 256) <= rounds(rtiles(4) * groups, 512)) wide = 8;
    // one tile of n workgroups, us: where each has a CU `one`; two workgroups of four waves share a CU in `two`, one-wave workgroups as many
    // as their LDS allows, a quarter longer for each more (f32 above 64 elements: one to a CU)
    const int row_bytes = a.dc <= 32 ? (bf16 ? 64 : 128) : a.dc <= 64 ? (bf16 ? 128 : 256) : a.dc <= 128 ? (bf16 ? 256 : 512) : (bf16 ? 512 : 1024);
    const double part = a.dc / 64.0 * a.kt / 64.0;
    const int per_cu = std::min(4, 160 * 1024 / (4 * a.kt * row_bytes));
    auto tile_us = [&](int waves, long long n) {
        if (waves == 1) {
            const double one = bf16 ? 0.8 + 0.6 * part : 5.0 * part;
            return rounds(n, 256 * per_cu) * one * (0.75 + 0.25 * std::min<long long>(per_cu, rounds(n, 256)));
        }
        const double one = waves == 8 ? 0.6 + 0.75 * part : bf16 ? 0.5 + 0.45 * part : 4.8 * part;
        if (waves == 8 || (!bf16 && a.dc > 64)) return rounds(n, 256) * one;
        const double two = bf16 ? (few ? 0.7 + 0.95 * part : 0.6 + 0.8 * part) : 7.5 * part;
        return n / 512 * two + (n % 512 == 0 ? 0.0 : n % 512 <= 256 ? one : two);
    };
    const double join_fixed_us = few ? 7.0 : 4.0;                                   // where latency counts also the launch on the host
    const double join_us = 4e-6 * 2 * B * Lq * (double)Hq * D / 4;                  // of one more split, at 4 TB/s
    double best = 0;
    a.splits = 0;
    auto consider = [&](int waves, int cs, double share) {
        const int rt = (int)rtiles(waves);
        for (int s = 1; s <= kMaxSplits && s <= tiles; ++s) {
            const int tps = (tiles + s - 1) / s, splits = (tiles + tps - 1) / tps;
            const double t = tile_us(waves, rt * groups * cs * splits) * share * (tps + 1.5) + (splits > 1 ? join_fixed_us + splits * (0.04 + join_us) : 0.0);
            if (a.splits == 0 || t < best) {
                best = t;
                a.waves = waves;
                a.rtiles = rt;
                a.cs = cs;
                a.splits = splits;
                a.tps = tps;
            }
        }
    };
    if (a.dc == 256) {
        if (!bf16) consider(4, 1, 1.0);
        consider(4, 2, bf16 ? 1.0 : 2.0 / 3);               // f32: scores and half of the results
    } else {
        consider(wide, 1, 1.0);
        if (few && (!bf16 || a.dc <= 64)) consider(1, 1, 1.0);
    }
    a.bytes = a.splits > 1 ? (size_t)a.splits * B * Lq * Hq * (D + 2) * 4 : 0;
    return a;
}

// MW: waves per SIMD the register budget is cut for.  Two hide each other's latencies where the tiles fill the GPU (D = 128, four waves:
// 804 us at one, 553 at two); one-wave workgroups run one to a SIMD, and f32 with more than 64 elements of o and q needs all 512 registers
template <bool BF16, int DC, int WAVES, int CS, bool WHOLE>
static int launch_attn_tile(const AttnK& p, hipStream_t stream) {
    constexpr int MW = (WAVES == 1 || (!BF16 && DC > 64)) ? 1 : 2;
    const unsigned long long blocks = (unsigned long long)p.rtiles * p.splits * p.B * p.Hk * CS;
    YOLO_REQUIRE(launchable(blocks, WAVES * 64), YOLO_ERR_UNSUPPORTED, "cross_attention: %llu workgroups are more than one launch takes", blocks);
    constexpr int kLds = 2 * AttnTile<BF16, DC>::TILE + 2 * AttnTile<BF16, DC>::KT * AttnTile<BF16, DC / CS>::ROW;
    if (kLds > 64 * 1024) {
        static std::atomic<bool> attr_done[16];   // setting the attribute twice is harmless, the flag only must not tear
        int dev = 0;
        YOLO_HIP_CHECK(hipGetDevice(&dev));
        if (dev >= 16 || !attr_done[dev]) {
            YOLO_HIP_CHECK(hipFuncSetAttribute((const void*)cross_attention_tile_kernel<BF16, DC, WAVES, MW, CS, WHOLE>,
                                               hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
            if (dev < 16) attr_done[dev] = true;
        }
    }
    hipLaunchKernelGGL((cross_attention_tile_kernel<BF16, DC, WAVES, MW, CS, WHOLE>), dim3((unsigned)blocks), dim3(WAVES * 64), kLds, stream, p);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}

// bf16 with few rows: whole weights, one or four waves
template <bool BF16, int DC>
static int launch_attn_dc(const AttnK& p, const AttnPlan& a, hipStream_t stream) {
    constexpr int CS = BF16 && DC == 256 ? 2 : 1;
    if constexpr (BF16) {
        if (a.few) {
            if constexpr (DC <= 64) {
                if (a.waves == 1) return launch_attn_tile<BF16, DC, 1, 1, true>(p, stream);
            }
            return launch_attn_tile<BF16, DC, 4, CS, true>(p, stream);
        }
        if constexpr (DC == 64 || DC == 96 || DC == 128) {
            if (a.waves == 8) return launch_attn_tile<BF16, DC, 8, 1, false>(p, stream);
        }
    } else {
        if constexpr (DC < 256) {
            if (a.waves == 1) return launch_attn_tile<BF16, DC, 1, 1, false>(p, stream);
        } else {
            if (a.cs == 2) return launch_attn_tile<BF16, DC, 4, 2, false>(p, stream);
        }
    }
    return launch_attn_tile<BF16, DC, 4, CS, false>(p, stream);
}

template <bool BF16>
static int launch_attn(const AttnK& p, const AttnPlan& a, hipStream_t stream) {
    int rc;
    switch (a.dc) {
        case 32: rc = launch_attn_dc<BF16, 32>(p, a, stream); break;
        case 64: rc = launch_attn_dc<BF16, 64>(p, a, stream); break;
        case 96: rc = launch_attn_dc<BF16, 96>(p, a, stream); break;
        case 128: rc = launch_attn_dc<BF16, 128>(p, a, stream); break;
        default: rc = launch_attn_dc<BF16, 256>(p, a, stream); break;
    }
    if (rc != YOLO_OK || p.splits == 1) return rc;
    const unsigned long long rows = (unsigned long long)p.B * p.Lq * p.Hq, blocks = p.splits > 8 ? rows : (rows * (p.D / 4) + 255) / 256;
    YOLO_REQUIRE(launchable(blocks, 256), YOLO_ERR_UNSUPPORTED, "cross_attention: %llu workgroups are more than one launch takes", blocks);
    if (p.splits > 8) hipLaunchKernelGGL(cross_attention_join_kernel<BF16>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(cross_attention_join_rows_kernel<BF16>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}

}  // namespace yolo

extern "C" size_t yolo_cross_attention_workspace_bytes(int dtype, int B, int Lq, int Lk, int Hq, int Hk, int D) {
    using namespace yolo;
    if ((dtype != YOLO_DTYPE_F32 && dtype != YOLO_DTYPE_BF16) || B <= 0 || Lq <= 0 || Lk <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk ||
        D <= 0 || D > 256 || D % 8 || (unsigned long long)B * Lq >= (1ull << 31) || Hq > 65536 || Lk > (1 << 30) ||
        (long long)Lq * (Hq / Hk) > (1ll << 30))
        return 0;
    return attn_plan(dtype, B, Lq, Lk, Hq, Hk, D).bytes;
}

extern "C" int yolo_cross_attention(int dtype, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                    const void* v, const int64_t* v_strides, const int32_t* key_lens, const uint8_t* key_mask,
                                    int B, int Lq, int Lk, int Hq, int Hk, int D, float scale, void* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    using namespace yolo;
    YOLO_REQUIRE(dtype == YOLO_DTYPE_F32 || dtype == YOLO_DTYPE_BF16, YOLO_ERR_ARG, "cross_attention: unknown dtype %d", dtype);
    YOLO_REQUIRE(B >= 0 && Lq >= 0 && Lk >= 0 && Hq > 0 && Hk > 0, YOLO_ERR_ARG, "cross_attention: bad size");
    YOLO_REQUIRE(Hq % Hk == 0, YOLO_ERR_SHAPE, "cross_attention: %d query heads do not share %d key heads evenly", Hq, Hk);
    YOLO_REQUIRE(D > 0 && D <= 256, YOLO_ERR_UNSUPPORTED, "cross_attention: head size %d, supported 1 to 256", D);
    if (B == 0 || Lq == 0) return YOLO_OK;
    YOLO_REQUIRE(q && q_strides && out && (Lk == 0 || (k && v && k_strides && v_strides)), YOLO_ERR_ARG, "cross_attention: null pointer");
    const int z = dtype == YOLO_DTYPE_BF16 ? 2 : 4;
    YOLO_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & (z - 1)) == 0 && ((uintptr_t)key_lens & 3) == 0,
                 YOLO_ERR_ARG, "cross_attention: a pointer is not aligned to its element");
    YOLO_REQUIRE((unsigned long long)B * Lq < (1ull << 31) && Hq <= 65536, YOLO_ERR_UNSUPPORTED, "cross_attention: B * Lq must be below 2^31, at most 65536 heads");
    YOLO_REQUIRE(std::isfinite(scale * 1.44269504f), YOLO_ERR_ARG, "cross_attention: scale must be finite");
    YOLO_REQUIRE(Lk <= (1 << 30), YOLO_ERR_UNSUPPORTED, "cross_attention: at most 2^30 keys");
    AttnK p;
    p.q = (const char*)q; p.k = (const char*)k; p.v = (const char*)v; p.out = (char*)out;
    p.lens = key_lens; p.mask = key_mask;
    p.qb = q_strides[0]; p.ql = q_strides[1]; p.qh = q_strides[2];
    p.kb = p.kl = p.kh = p.vb = p.vl = p.vh = 0;
    if (Lk) {
        p.kb = k_strides[0]; p.kl = k_strides[1]; p.kh = k_strides[2];
        p.vb = v_strides[0]; p.vl = v_strides[1]; p.vh = v_strides[2];
    }
    p.B = B; p.Lq = Lq; p.Lk = Lk; p.Hq = Hq; p.Hk = Hk; p.D = D; p.G = Hq / Hk; p.scale = scale;
    p.part = nullptr; p.ml = nullptr; p.q_and = ~0u; p.q_xor = 0; p.scale2 = 0.f; p.rtiles = 0; p.splits = 1; p.tps = 0;
    // the matrix-core kernels read whole 16-byte pieces of rows and hold the rows of a head group in 32 bits
    bool fast = Lk > 0 && D % 8 == 0 && aligned16(out) && (long long)Lq * p.G <= (1ll << 30);
    const void* base[3] = {q, k, v};
    const int64_t* st[3] = {q_strides, k_strides, v_strides};
    for (int i = 0; fast && i < 3; ++i)
        fast = aligned16(base[i]) && st[i][0] * z % 16 == 0 && st[i][1] * z % 16 == 0 && st[i][2] * z % 16 == 0;
    if (fast) {
        const AttnPlan a = attn_plan(dtype, B, Lq, Lk, Hq, Hk, D);
        p.rtiles = a.rtiles; p.splits = a.splits; p.tps = a.tps;
        p.scale2 = scale == 0.f ? 1.44269504f : std::fabs(scale) * 1.44269504f;
        p.q_and = scale == 0.f ? 0u : ~0u;
        p.q_xor = scale < 0.f ? (dtype == YOLO_DTYPE_BF16 ? 0x80008000u : 0x80000000u) : 0u;
        if (a.splits > 1) {
            YOLO_REQUIRE(workspace && workspace_bytes >= a.bytes && aligned16(workspace), YOLO_ERR_WORKSPACE,
                         "cross_attention: workspace of %zu bytes (16-byte aligned) needed, got %zu", a.bytes, workspace ? workspace_bytes : (size_t)0);
            p.part = (float*)workspace;
            p.ml = (float2*)(p.part + (size_t)a.splits * B * Lq * Hq * D);
        }
        return dtype == YOLO_DTYPE_BF16 ? launch_attn<true>(p, a, (hipStream_t)stream) : launch_attn<false>(p, a, (hipStream_t)stream);
    }
    const unsigned long long blocks = ((unsigned long long)B * Lq * Hq + 3) / 4;
    YOLO_REQUIRE(launchable(blocks, 256), YOLO_ERR_UNSUPPORTED, "cross_attention: %llu workgroups are more than one launch takes", blocks);
    if (dtype == YOLO_DTYPE_BF16) hipLaunchKernelGGL(cross_attention_general_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(cross_attention_general_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}
