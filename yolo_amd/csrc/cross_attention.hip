// yolo_cross_attention: o = softmax(scale * q k^T) v over the kept keys of another sequence, query heads in groups that share a
// key / value head.
//
// Mathematics: one pass over the keys with the running maximum m and sum l of the softmax: with m' = max(m, max s),
// o <- o exp(m - m') + sum exp(s - m') v and l likewise, result o / l.  Scores, m, l and o are f32.  A key is kept when its
// index is below key_lens[b] and its key_mask byte is set; what is not kept is never multiplied (its score is replaced, its
// value row not used), so that infinities and NaN there stay out.  A row without a kept key is zero.
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

}  // namespace yolo

extern "C" size_t yolo_cross_attention_workspace_bytes(int dtype, int B, int Lq, int Lk, int Hq, int Hk, int D) {
    (void)dtype; (void)B; (void)Lq; (void)Lk; (void)Hq; (void)Hk; (void)D;
    return 0;
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
    (void)workspace; (void)workspace_bytes;
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
    const unsigned long long blocks = ((unsigned long long)B * Lq * Hq + 3) / 4;
    YOLO_REQUIRE(blocks < (1ull << 31), YOLO_ERR_UNSUPPORTED, "cross_attention: more than 2^33 rows");
    if (dtype == YOLO_DTYPE_BF16) hipLaunchKernelGGL(cross_attention_general_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(cross_attention_general_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
    YOLO_HIP_CHECK(hipGetLastError());
    return YOLO_OK;
}
