// yolo_qk_norm_rope: the norms of queries and keys for each head and the rotation by position, both sides in one launch.
//
// Mathematics, per (token, head) row x of D elements:  h = x / sqrt(mean(x^2) + eps) * w;  pair i of the first R = rotary_dim
// elements, (h_i, h_{i+R/2}) or, interleaved, (h_2i, h_2i+1), is turned by the angle a = position * frequency_i:
// (u, v) -> (u cos a - v sin a, u sin a + v cos a).  With two axes (row, column of a map cell) the first half of the pairs
// turns by the first coordinate, the second half by the second.
// Sum of squares, norm and rotation in f32, one rounding at the store; the angle is formed and reduced to a fraction of a turn
// in f64 (position 10^6 at frequency 1 leaves 10^-10 of an angle; in f32 it would leave 0.06), sine and cosine in f32.
#include "layer_common.h"

namespace yolo {

struct RopeSide {
    const char* x;
    const void* w;             // norm weight [D] or nullptr (ones)
    const void* pos;           // [L, A] or [B, L, A], int32 or int64
    char* out;                 // [B, L, H, D] packed
    long long sb, sl, sh;      // element strides of x
    int L, H;
    int tokens;                // B * L
    int tpb;                   // tokens per workgroup
    int pos_batched;
};

struct RopeK {
    RopeSide side[2];
    unsigned blocks0;          // workgroups of side 0
    int D, R, axes, interleaved, w_bf16, pos64;
    const double* freq;        // [R / 2] radians per position, nullptr: no rotation
    float eps;
};

constexpr int kRopeTable = 512;     // (cos, sin) pairs a workgroup computes, two a thread, and keeps in LDS; a token has at most 128

// cos / sin of every (token, pair) of this workgroup and the norm weights -> LDS
__device__ __forceinline__ void rope_tables(const RopeK& p, const RopeSide& s, int t0, int nt, float2* cs, float* wt) {
    for (int d = threadIdx.x; d < p.D; d += 256) wt[d] = s.w ? load_param(s.w, p.w_bf16, d) : 1.0f;
    if (!p.freq) return;
    const int half = p.R >> 1, per_axis = half / p.axes;
    for (int e = threadIdx.x; e < nt * half; e += 256) {
        const int t = t0 + e / half, i = e % half;
        const long long pi = (long long)(s.pos_batched ? t : t % s.L) * p.axes + i / per_axis;
        const double pos = p.pos64 ? (double)((const long long*)s.pos)[pi] : (double)((const int*)s.pos)[pi];
        double turn = pos * p.freq[i] * 0.15915494309189535;       // radians -> turns
        turn -= rint(turn);
        float sn, cn;
        sincospif((float)(2.0 * turn), &sn, &cn);
        cs[e] = make_float2(cn, sn);
    }
}

// Any D <= 256, any rotary_dim, any alignment: one wave per row, lane holds elements lane + 64 i, partners meet through LDS.
template <bool BF16>
__global__ __launch_bounds__(256) void qk_norm_rope_general_kernel(RopeK p) {
    typedef typename Elem<BF16>::type T;
    __shared__ float2 cs[kRopeTable];
    __shared__ float wt[256];
    __shared__ float row[4][256];
    const bool second = blockIdx.x >= p.blocks0;
    const RopeSide& s = p.side[second];
    const int t0 = (int)(blockIdx.x - (second ? p.blocks0 : 0)) * s.tpb;
    const int nt = min(s.tpb, s.tokens - t0);
    rope_tables(p, s, t0, nt, cs, wt);
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = p.R >> 1;
    const int rows = nt * s.H;
    for (int r0 = 0; r0 < rows; r0 += 4) {
        const int r = r0 + wave;
        const bool in = r < rows;
        const int tl = in ? r / s.H : 0, h = in ? r % s.H : 0, t = t0 + tl;
        const T* x = (const T*)s.x + (long long)(t / s.L) * s.sb + (long long)(t % s.L) * s.sl + (long long)h * s.sh;
        float v[4], ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            v[i] = in && d < p.D ? load_f32(x + d) : 0.f;
            ss = __builtin_fmaf(v[i], v[i], ss);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        const float rs = 1.0f / sqrtf(ss / (float)p.D + p.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (d < p.D) row[wave][d] = v[i] * rs * wt[d];
        }
        __syncthreads();
        if (in) {
            T* o = (T*)s.out + ((long long)t * s.H + h) * p.D;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = lane + 64 * i;
                if (d >= p.D) continue;
                float y = row[wave][d];
                if (p.freq && d < p.R) {
                    const bool hi = p.interleaved ? (d & 1) : d >= half;
                    const int pair = p.interleaved ? d >> 1 : (hi ? d - half : d);
                    const float z = row[wave][p.interleaved ? d ^ 1 : (hi ? d - half : d + half)];
                    const float2 c = cs[tl * half + pair];
                    y = hi ? __builtin_fmaf(z, c.y, y * c.x) : __builtin_fmaf(-z, c.y, y * c.x);
                }
                o[d] = (T)y;
            }
        }
        __syncthreads();
    }
}

// The usual layout: D and rotary_dim whole pairs of 16-byte pieces, aligned rows.  A lane holds two pieces whose elements are each
// other's partners - elements c P .. and R/2 + c P .. of a row, or neighbours if interleaved or past rotary_dim - so that the rotation
// needs no exchange; LPR = D / (2 pieces) lanes, rounded up to a power of two, make a row, and its sum of squares is log2(LPR) lane
// exchanges.
// Bandwidth bounds it: a workgroup issues its first row loads before it computes the table (one sine / cosine per thread or so,
// shared by all heads of a token).
template <bool BF16>
__device__ __forceinline__ void unpack_piece(u32x4 v, float* f) {
    if constexpr (BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = bf16_lo(v[j]);
            f[2 * j + 1] = bf16_hi(v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(v[j]);
    }
}

template <bool BF16>
__device__ __forceinline__ u32x4 pack_piece(const float* f) {
    u32x4 v;
    if constexpr (BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = pack_bf16(f[2 * j], f[2 * j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __float_as_uint(f[j]);
    }
    return v;
}

template <bool BF16, int LPR, bool IL>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeK p) {
    typedef typename Elem<BF16>::type T;
    constexpr int P = Elem<BF16>::kPiece, RPP = 256 / LPR;     // rows a pass of the workgroup covers
    __shared__ float2 cs[kRopeTable];
    __shared__ float wt[256];
    const bool second = blockIdx.x >= p.blocks0;
    const RopeSide& s = p.side[second];
    const int t0 = (int)(blockIdx.x - (second ? p.blocks0 : 0)) * s.tpb;
    const int nt = min(s.tpb, s.tokens - t0), rows = nt * s.H;
    const int c = threadIdx.x % LPR, rw = threadIdx.x / LPR;
    const bool lane_in = c * 2 * P < p.D;                       // D / (2 P) lanes of the LPR hold pieces
    const bool turned = c * 2 * P < p.R;                        // the lanes before the first that is not hold R elements
    const int da = IL || !turned ? 2 * c * P : c * P, db = IL || !turned ? da + P : da + p.R / 2;
    u32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    int tl = 0, h = 0;
    auto load = [&](int r) {
        a = b = u32x4{0, 0, 0, 0};
        if (r >= rows || !lane_in) return;
        tl = r / s.H;
        h = r - tl * s.H;
        const int t = t0 + tl, bi = t / s.L;
        const T* x = (const T*)s.x + bi * s.sb + (t - bi * s.L) * s.sl + h * s.sh;
        a = *(const u32x4*)(x + da);
        b = *(const u32x4*)(x + db);
    };
    load(rw);
    rope_tables(p, s, t0, nt, cs, wt);
    __syncthreads();
    float wa[P], wb[P];
    if (lane_in) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            wa[j] = wt[da + j];
            wb[j] = wt[db + j];
        }
    }
    for (int r = rw; r < rows + rw; r += RPP) {                 // every lane of a wave makes the same trips: r - rw is uniform
        float u[P], v[P], ss = 0.f;
        unpack_piece<BF16>(a, u);
        unpack_piece<BF16>(b, v);
        const int tc = tl, hc = h;
        const bool in = r < rows && lane_in;
        if (r + RPP < rows) load(r + RPP);                      // the next row is on its way while this one is computed
#pragma unroll
        for (int j = 0; j < P; ++j) ss = __builtin_fmaf(u[j], u[j], __builtin_fmaf(v[j], v[j], ss));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        if (!in) continue;
        const float rs = 1.0f / sqrtf(ss / (float)p.D + p.eps);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            u[j] *= rs * wa[j];
            v[j] *= rs * wb[j];
        }
        if (turned) {
            const float2* t = cs + tc * (p.R / 2) + c * P;      // pairs c P .. c P + P - 1 in either layout
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const float2 w = t[j];
                float& x = IL ? (2 * j < P ? u[(2 * j) % P] : v[(2 * j) % P]) : u[j];
                float& y = IL ? (2 * j < P ? u[(2 * j) % P + 1] : v[(2 * j) % P + 1]) : v[j];
                const float x0 = x, y0 = y;
                x = __builtin_fmaf(-y0, w.y, x0 * w.x);
                y = __builtin_fmaf(x0, w.y, y0 * w.x);
            }
        }
        T* o = (T*)s.out + ((long long)(t0 + tc) * s.H + hc) * p.D;
        *(u32x4*)(o + da) = pack_piece<BF16>(u);
        *(u32x4*)(o + db) = pack_piece<BF16>(v);
    }
}

template <bool BF16, int LPR>
static void launch_rope_rows(const RopeK& p, unsigned blocks, hipStream_t stream) {
    if (p.interleaved) hipLaunchKernelGGL((qk_norm_rope_kernel<BF16, LPR, true>), dim3(blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<BF16, LPR, false>), dim3(blocks), dim3(256), 0, stream, p);
}

template <bool BF16>
static void launch_rope(const RopeK& p, int lpr, unsigned blocks, hipStream_t stream) {
    switch (lpr) {
        case 1: launch_rope_rows<BF16, 1>(p, blocks, stream); break;
        case 2: launch_rope_rows<BF16, 2>(p, blocks, stream); break;
        case 4: launch_rope_rows<BF16, 4>(p, blocks, stream); break;
        case 8: launch_rope_rows<BF16, 8>(p, blocks, stream); break;
        case 16: launch_rope_rows<BF16, 16>(p, blocks, stream); break;
        case 32:
            if constexpr (!BF16) {                              // a bf16 row is at most 16 pairs of pieces
                launch_rope_rows<BF16, 32>(p, blocks, stream);
                break;
            }
            [[fallthrough]];
        default: hipLaunchKernelGGL(qk_norm_rope_general_kernel<BF16>, dim3(blocks), dim3(256), 0, stream, p);
    }
}

}  // namespace yolo

extern "C" int yolo_qk_norm_rope(int dtype, int B, int D, const void* q, const int64_t* q_strides, int Lq, int Hq,
                                 const void* q_weight, const void* q_positions, void* q_out, const void* k,
                                 const int64_t* k_strides, int Lk, int Hk, const void* k_weight, const void* k_positions,
                                 void* k_out, int weight_dtype, const double* frequencies, int rotary_dim, int axes,
                                 int positions_int64, int q_positions_batched, int k_positions_batched, int interleaved,
                                 float eps, void* stream) {
    using namespace yolo;
    YOLO_REQUIRE(dtype == YOLO_DTYPE_F32 || dtype == YOLO_DTYPE_BF16, YOLO_ERR_ARG, "qk_norm_rope: unknown dtype %d", dtype);
    YOLO_REQUIRE(weight_dtype == YOLO_DTYPE_F32 || weight_dtype == YOLO_DTYPE_BF16, YOLO_ERR_ARG, "qk_norm_rope: unknown weight dtype %d", weight_dtype);
    YOLO_REQUIRE(B >= 0 && Lq >= 0 && Lk >= 0 && Hq > 0 && (!k || Hk > 0), YOLO_ERR_ARG, "qk_norm_rope: bad size");
    YOLO_REQUIRE(D > 0 && D <= 256, YOLO_ERR_UNSUPPORTED, "qk_norm_rope: head size %d, supported 1 to 256", D);
    YOLO_REQUIRE(eps > 0.f, YOLO_ERR_ARG, "qk_norm_rope: eps must be positive");
    if (frequencies) {
        YOLO_REQUIRE(rotary_dim > 0 && rotary_dim <= D && rotary_dim % 2 == 0, YOLO_ERR_ARG, "qk_norm_rope: rotary_dim %d must be even and within the head size %d", rotary_dim, D);
        YOLO_REQUIRE((axes == 1 || axes == 2) && rotary_dim / 2 % axes == 0, YOLO_ERR_ARG, "qk_norm_rope: %d pairs do not split over %d axes", rotary_dim / 2, axes);
    } else {
        rotary_dim = 0;
        axes = 1;
    }
    RopeK p;
    p.D = D; p.R = rotary_dim; p.axes = axes; p.interleaved = interleaved != 0; p.w_bf16 = weight_dtype == YOLO_DTYPE_BF16;
    p.pos64 = positions_int64 != 0; p.freq = frequencies; p.eps = eps;
    const int z = dtype == YOLO_DTYPE_BF16 ? 2 : 4;
    const int piece = 16 / z;
    // lanes per row of the register kernel, 0: general kernel
    int lpr = 0;
    if (D % (2 * piece) == 0 && rotary_dim % (2 * piece) == 0)
        for (lpr = 1; lpr * 2 * piece < D;) lpr *= 2;
    for (int i = 0; i < 2 && lpr; ++i) {
        const int64_t* st = i ? k_strides : q_strides;
        const void* x = i ? k : q;
        if (!x || !st) continue;
        if (!aligned16(x) || !aligned16(i ? k_out : q_out) || st[0] * z % 16 || st[1] * z % 16 || st[2] * z % 16) lpr = 0;
    }
    unsigned long long blocks[2] = {0, 0};
    for (int i = 0; i < 2; ++i) {
        RopeSide& s = p.side[i];
        s.x = (const char*)(i ? k : q); s.w = i ? k_weight : q_weight; s.pos = i ? k_positions : q_positions;
        s.out = (char*)(i ? k_out : q_out);
        s.L = i ? Lk : Lq; s.H = i ? Hk : Hq;
        s.pos_batched = i ? k_positions_batched : q_positions_batched;
        s.sb = s.sl = s.sh = 0; s.tokens = 0; s.tpb = 1;
        const bool absent = i ? !k || Lk == 0 : Lq == 0;
        if (absent || B == 0) continue;
        const int64_t* st = i ? k_strides : q_strides;
        YOLO_REQUIRE(s.x && s.out && st, YOLO_ERR_ARG, "qk_norm_rope: null pointer");
        YOLO_REQUIRE(!frequencies || s.pos, YOLO_ERR_ARG, "qk_norm_rope: frequencies without positions");
        YOLO_REQUIRE((((uintptr_t)s.x | (uintptr_t)s.out) & (z - 1)) == 0, YOLO_ERR_ARG, "qk_norm_rope: a pointer is not aligned to its element");
        YOLO_REQUIRE((long long)B * s.L < (1ll << 31) && s.H <= 65536, YOLO_ERR_UNSUPPORTED, "qk_norm_rope: B * L must be below 2^31, at most 65536 heads");
        s.sb = st[0]; s.sl = st[1]; s.sh = st[2];
        s.tokens = B * s.L;
        s.tpb = (lpr ? 2 * 256 / lpr : 32) / s.H;              // two rows for every lane group
        if (s.tpb < 1) s.tpb = 1;
        if (p.R && s.tpb > kRopeTable / (p.R / 2)) s.tpb = kRopeTable / (p.R / 2);
        blocks[i] = ((unsigned long long)s.tokens + s.tpb - 1) / s.tpb;
    }
    const unsigned long long total = blocks[0] + blocks[1];
    if (total == 0) return YOLO_OK;
    YOLO_REQUIRE(launchable(total, 256), YOLO_ERR_UNSUPPORTED, "qk_norm_rope: %llu workgroups are more than one launch takes", total);
    p.blocks0 = (unsigned)blocks[0];
    if (dtype == YOLO_DTYPE_BF16) launch_rope<true>(p, lpr, (unsigned)total, (hipStream_t)stream);
    else launch_rope<false>(p, lpr, (unsigned)total, (hipStream_t)stream);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}
