// The chunked delta rule with kept states for heads of 128 values (or a multiple of 64): chunks of 64 tokens on tcgen05.  The algebra, the
// pieces and the scales are those of gdn_prefill.cu, with 64 for 16:
//
//     U = T (V - diag(e) K S0),  O = M U + diag(e) Q S0,  S = e_64 S0 + K^T diag(exp(c_64 - c_j)) U
//
// prep   a CTA per chunk and head: T and M, what needs no state.  Gram products of 16 x 16 blocks on mma.sync; of the triangular inverse the
//        blocks on the diagonal by substitution in float32, those below it as products of blocks on the tensor cores, each factor in two
//        TF32 pieces.  Both leave as fp16 pieces in the layout that the tensor core reads, the blocks above the diagonal left out: 16,912
//        bytes a chunk (22,032 with the second piece of M, for fp16).  For bf16 the second piece of M's rows waits in the
//        rows of o that it makes, 128 bytes of each, until the chunk's outputs go there: four CTAs of prep fit an SM so (with it in
//        the workspace three, as for fp16: 285 us for 64 x 2,048 tokens instead of 265), and walk loads it by TMA.
// walk   a CTA per head and 128 value columns.  The values are the 128 lanes of tensor memory: S^T, W^T, U^T and D^T are operands that
//        lie there as pieces, K, Q, T and M come from shared memory.  The state itself stays in registers: a value column's keys in two
//        threads (eight warps), rounded by float32 FMAs; per chunk its pieces go to tensor memory and the product K^T D comes back.
//        Four more warps write the outputs, one issues the products, one the copies (TMA, a chunk or two ahead), two turn K and Q into
//        scaled fp16 in place.
//
// A chunk is a chain: pieces of S -> K S0 -> W -> T W -> D -> K^T D -> S.  Q S0 and M U run beside it, and the outputs of a chunk are
// written while the next one's first product runs.
//
// What bounds it.  64 sequences of 2,048 tokens, 6 heads of 128 x 128, bf16: prep 265 us and walk 420 by themselves, 648 for the call, for
// 862 MB that have to move (131 us at the rate of a plain copy) and 0.16 TFLOP of the walk's products (97 us at cuBLAS's bf16 rate).  The
// walk is bound by its chain: a chunk takes 2.8 us (4.2 with all SMs at work), of which the three products that it waits for are about 0.9;
// cutting into pieces, the ways through tensor memory and shared memory and the meetings of threads are the rest.  A CTA takes all columns of
// tensor memory and nearly all shared memory of an SM, so no second chain fills the gaps (384 chains on 148 SMs: three waves).  An
// instruction that is not in the cache costs most beside that, which is why the loops below are rolled where they can be.  prep is a row of short phases between barriers, four CTAs of four warps on
// an SM (issue slots 46 % used, DRAM 20 %): loads 63 us, Gram products 39, scalars and masks 46, the diagonal's inverses 17, the products of
// blocks 40, T's pieces 22, the copy out 11, M's second piece 20.
// One sequence of 16,384 tokens, 6 heads: prep 38 us, the two walks of its segments 99 and 89, the join 30, by themselves; the kernels overlap
// where one drains: 241 us for the call, 34 for one of 321 tokens with heads of 64 x 128.
#include "gdn_pieces.cuh"
#include "gdn_seq.cuh"
#include "tc_ptx.cuh"
#include "tma_utils.cuh"

#include <type_traits>

namespace sb {
namespace {

using namespace tc;

constexpr int CT = 64;                                           // tokens of a chunk
constexpr int TV = 128;                                          // value columns of a CTA
// A triangular 64 x 64 fp16 matrix [i][j], j in steps of 16: step kk holds rows 16 kk .. 63, 32 bytes each, in core matrices of 8 rows x 16
// bytes (rows 16 bytes apart, the two of a step's 16 columns 128 apart, the next 8 rows 256 apart): (i, j) at
// tri_at(i, j) = tri_step(j / 16) + (r / 8) 256 + (j / 8 % 2) 128 + (r % 8) 16 + (j % 8) 2, r = i - 16 (j / 16).
constexpr int TRI_BYTES = 5120;
__host__ __device__ constexpr int tri_step(int kk) { return 32 * (64 * kk - 8 * kk * (kk - 1)); }
// workspace of a chunk and head: T hi | T lo | M hi | (M lo, fp16 calls) | six arrays of 64 floats | e_64, T's scale, the largest ER, DK's scale
template <bool LO_WS> struct Ws {
    static constexpr int T = 0, TL = TRI_BYTES, M = 2 * TRI_BYTES, ML = 3 * TRI_BYTES, SC = (LO_WS ? 4 : 3) * TRI_BYTES;
    static constexpr int ER = SC, EQ = SC + 256, DK = SC + 512, OM = SC + 768, KS = SC + 1024, QS = SC + 1280, E64 = SC + 1536;
    static constexpr int BYTES = SC + 1552;
};

__device__ int g_prefill_status = 0;                             // 1 + role whose wait gave up

// 128-byte rows, 16-byte pieces swizzled by the row: what SWIZZLE_128B reads
__device__ __forceinline__ uint32_t sw128(int row, int piece) { return uint32_t(row * 128 + ((piece ^ (row & 7)) << 4)); }


// Chunks of sequence n stand at [start / 64 + n, .. + ceil(length / 64)) of the workspace: never over those of n + 1, for any lengths.
__device__ __forceinline__ int first_chunk(const SeqRows& r, int n) { return r.start / CT + n; }

// ---------------------------------------------------------------------------------------------------- what needs no state
template <int DK, bool LO_WS> struct PrepSmem {
    static constexpr int TILES = 2 * CT * DK * 2, IMAGES = Ws<LO_WS>::BYTES, LP = CT + 4;
    static constexpr int X_AT = (IMAGES + 15) / 16 * 16, BOTH = X_AT + CT * LP * 4;
    __align__(1024) uint8_t a[TILES > BOTH ? TILES : BOTH];      // K and Q as they are, then what leaves and, behind it, X = (I + L)^-1
    __align__(16) float l[CT * LP];
    double cum[CT], low[CT];                                     // cumulative decay, and its least value so far
    float beta[CT], kk[CT], qq[CT], top[4];
    float row[3][CT], col[CT];                                   // decay of a token since the end of block b; of a block's end since a token
    float erm[2], dkm[2];                                        // the largest ER and DK of 32 tokens
    float bk[CT], rk[CT], rq[CT];                                // beta / |k|, 1 / |k|, scale / |q| and M's row scale
};

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d += A B of two 16 x 16 blocks (pitch P) in shared memory, to 22 bits: hi and lo are eleven bits each
template <int P> __device__ __forceinline__ void block_product(float (&d)[2][4], const float* A, const float* B, int g, int t) {
    auto split = [](float v, uint32_t& hi, uint32_t& lo) {
        hi = __float_as_uint(v) & 0xffffe000u;
        lo = __float_as_uint(v - __uint_as_float(hi)) & 0xffffe000u;
    };
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split(A[(g + 8 * (i & 1)) * P + k + t + 4 * (i >> 1)], ah[i], al[i]);
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            uint32_t bh[2], bl[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) split(B[(k + t + 4 * i) * P + 8 * ni + g], bh[i], bl[i]);
            mma_tf32(d[ni], al, bh[0], bh[1]);
            mma_tf32(d[ni], ah, bl[0], bl[1]);
            mma_tf32(d[ni], ah, bh[0], bh[1]);
        }
    }
}
template <int P> __device__ __forceinline__ void block_store(float* D, const float (&d)[2][4], float sign, int g, int t) {
#pragma unroll
    for (int ni = 0; ni < 2; ++ni)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(D + (g + 8 * h) * P + 8 * ni + 2 * t) = make_float2(sign * d[ni][2 * h], sign * d[ni][2 * h + 1]);
}

template <typename T> constexpr bool M_LO_IN_WS = std::is_same<T, __half>::value;     // M's second piece: in the workspace, or in o's rows
template <typename T, int DK>
__global__ void __launch_bounds__(128, M_LO_IN_WS<T> ? 3 : 4) gdn_prefill_tc_prep_kernel(const shvk_gdn_seq_args a, uint8_t* __restrict__ ws) {
    constexpr bool LO_WS = M_LO_IN_WS<T>;
    using W = Ws<LO_WS>;
    using Sm = PrepSmem<DK, LO_WS>;
    constexpr int LP = Sm::LP;
    extern __shared__ uint8_t prep_raw[];
    Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(prep_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    last_is_done();
    next_may_start();                                            // (behind the wait: the walk reads where sequences lie before its own)
    const int chunk = int(blockIdx.x / unsigned(a.HV)), head = int(blockIdx.x % unsigned(a.HV)), khead = head / (a.HV / a.HK);
    int n = 0;                                                   // the last sequence whose first chunk is not behind this one
    for (int lo = 0, hi = a.n_seq - 1; lo <= hi;) {
        const int mid = (lo + hi) >> 1;
        if (first_chunk(SeqRows(a.seq_start, mid, int(a.n_tokens)), mid) <= chunk) { n = mid; lo = mid + 1; } else hi = mid - 1;
    }
    const SeqRows rows(a.seq_start, n, int(a.n_tokens));
    const int ahead = chunk - first_chunk(rows, n);
    if (ahead < 0 || (long long)ahead * CT >= rows.end - rows.start) return;       // no chunk of any sequence stands here
    const int t0 = rows.start + ahead * CT, left = rows.end - t0;
    uint8_t* kt = sm.a;
    uint8_t* qt = sm.a + CT * DK * 2;
    float* xs = reinterpret_cast<float*>(sm.a + Sm::X_AT);
    const uint32_t k_s = smem_u32(kt), q_s = smem_u32(qt);
    {
        const T* Q = static_cast<const T*>(a.q) + t0 * a.ldq + khead * DK;
        const T* K = static_cast<const T*>(a.k) + t0 * a.ldk + khead * DK;
#pragma unroll
        for (int i = 0; i < CT * DK / 8 / 128; ++i) {
            const int v = tid + 128 * i, row = v / (DK / 8), p = v % (DK / 8), has = row < left ? 16 : 0;
            const uint32_t off = (p >> 3) * (CT * 128) + sw128(row, p & 7);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(k_s + off), "l"(has ? static_cast<const void*>(K + row * a.ldk + p * 8) : ws), "r"(has) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_s + off), "l"(has ? static_cast<const void*>(Q + row * a.ldq + p * 8) : ws), "r"(has) : "memory");
        }
    }
    if (warp == 0) {                                             // cumulative decays in double: their differences are exponents
        double v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int tok = 2 * lane + e;
            const float g = tok < left ? a.g[(t0 + tok) * a.ldgb + head] : 0.0f;
            v[e] = g < -1000.0f ? -1000.0f : g;                  // exp(-1000) = 0, and no difference of two infinities (NaN stays)
        }
        double s = v[0] + v[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += up;
        }
        const double until = __shfl_up_sync(0xffffffffu, s, 1);
        v[0] += lane ? until : 0.0;
        v[1] += v[0];
        double mm = fmin(v[0], v[1]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, mm, o);
            if (lane >= o) mm = fmin(mm, up);
        }
        const double before = __shfl_up_sync(0xffffffffu, mm, 1);
        sm.cum[2 * lane] = v[0];
        sm.cum[2 * lane + 1] = v[1];
        sm.low[2 * lane] = lane ? fmin(before, v[0]) : v[0];
        sm.low[2 * lane + 1] = lane ? fmin(before, fmin(v[0], v[1])) : fmin(v[0], v[1]);
    } else if (tid >= 64) {
        const int tok = tid - 64;
        sm.beta[tok] = tok < left ? a.beta[(t0 + tok) * a.ldgb + head] : 0.0f;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // ---------------------------------------------------------------- Gram products of the blocks (bi, bj), bj <= bi; the first is (warp, warp)
    const int g = lane >> 2, t = lane & 3, lm = lane >> 3, lr = lane & 7;
    const int blocks = warp < 2 ? 3 : 2;
    auto bi_of = [&](int b) { return b == 0 ? warp : b == 1 ? (warp == 0 ? 3 : warp == 1 ? 1 : 2) : 3; };
    auto bj_of = [&](int b) { return b == 0 ? warp : b == 1 ? (warp == 3 ? 1 : 0) : warp == 0 ? 1 : 2; };     // w0 00 30 31, w1 11 10 32, w2 22 20, w3 33 21
    float kk[3][2][4] = {}, qk[3][2][4] = {};
    {
        float qq[2][4] = {};
#pragma unroll
        for (int b = 0; b < 3; ++b) {
            if (b >= blocks) break;
            const int ri = 16 * bi_of(b) + (lm & 1) * 8 + lr, rj = 16 * bj_of(b) + (lm & 1) * 8 + lr;
#pragma unroll
            for (int p = 0; p < DK / 16; ++p) {
                const uint32_t half = (p >> 2) * (CT * 128), piece = 2 * (p & 3) + (lm >> 1);
                uint32_t ki[4], qi[4], kj[4];
                ldsm4(q_s + half + sw128(ri, piece), qi);
                ldsm4(k_s + half + sw128(ri, piece), ki);
                if (b > 0) ldsm4(k_s + half + sw128(rj, piece), kj);
#pragma unroll
                for (int ni = 0; ni < 2; ++ni) {
                    const uint32_t b0 = b > 0 ? kj[ni] : ki[ni], b1 = b > 0 ? kj[ni + 2] : ki[ni + 2];
                    mma16<T>(kk[b][ni], ki, b0, b1);
                    mma16<T>(qk[b][ni], qi, b0, b1);
                    if (b == 0) mma16<T>(qq[ni], qi, qi[ni], qi[ni + 2]);
                }
            }
        }
        if ((g >> 1) == t) {                                     // the diagonal: [ni][2 ni + e] of lane (g, t) is entry (8 ni + g, 8 ni + 2 t + e)
            const int e = g & 1;
            sm.kk[16 * warp + g] = e ? kk[0][0][1] : kk[0][0][0];
            sm.kk[16 * warp + 8 + g] = e ? kk[0][1][3] : kk[0][1][2];
            sm.qq[16 * warp + g] = e ? qq[0][1] : qq[0][0];
            sm.qq[16 * warp + 8 + g] = e ? qq[1][3] : qq[1][2];
        }
    }
    __syncthreads();                                             // norms are there; K and Q are read
    uint8_t* out = sm.a;
    auto outf = [&](int at) { return reinterpret_cast<float*>(out + at); };
    const int tok = tid & 63;
    const double cs = sm.cum[tok], last = sm.cum[CT - 1];
    const float k2 = sm.kk[tok], rk = a.l2norm ? 1.0f / sqrtf(k2 + 1e-6f) : 1.0f;
    {
        const float most = warp_max(rk * sqrtf(k2));             // the longest key (of 32 tokens)
        if (lane == 0 && warp < 2) sm.top[warp] = most;
    }
    // exp(c_i - c_j) of a block below the diagonal is exp(c_i - c_e) exp(c_e - c_j), e the last token of j's block.
    if (tid < CT) {
        sm.col[tok] = expf(float(sm.cum[tok | 15] - cs));
        sm.row[0][tok] = expf(float(cs - sm.cum[15]));
    } else {
        sm.row[1][tok] = expf(float(cs - sm.cum[31]));
        sm.row[2][tok] = expf(float(cs - sm.cum[47]));
    }
    __syncthreads();
    if (tid < CT) {
        const int ke = clampi(exponent_of(sqrtf(k2)), 27, 227);
        const float e = expf(float(cs)), d = expf(float(last - cs)), kap = rk * pow2_biased(ke + 1);     // rk / ks
        sm.rk[tok] = rk;
        sm.bk[tok] = sm.beta[tok] * rk;
        outf(W::KS)[tok] = pow2_biased(253 - ke);                // |ks k| < 1
        outf(W::ER)[tok] = e * kap;
        outf(W::DK)[tok] = d * kap;                              // to be scaled to at most one
        const float em = warp_max(e * kap <= 3.402823466e38f ? e * kap : 0.0f), dm = warp_max(d * kap);
        if (lane == 0) { sm.erm[warp] = em; sm.dkm[warp] = dm; }
    } else {
        const float q2 = sm.qq[tok], rq = a.scale * (a.l2norm ? 1.0f / sqrtf(q2 + 1e-6f) : 1.0f);
        const int qe = clampi(exponent_of(sqrtf(q2)), 27, 227);
        outf(W::QS)[tok] = pow2_biased(253 - qe);
        outf(W::EQ)[tok] = expf(float(cs)) * (rq * pow2_biased(qe + 1));
        // a row of M is at most |q| |k| times its largest decay
        const float most = fabsf(rq) * sqrtf(q2) * fmaxf(sm.top[0], sm.top[1]) * expf(float(cs - sm.low[tok]));
        const int me = clampi(exponent_of(most), 27, 227);
        outf(W::OM)[tok] = pow2_biased(me + 1);
        sm.rq[tok] = rq * pow2_biased(253 - me);
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 3; ++b) {
        if (b >= blocks) break;
        const int bi = bi_of(b), bj = bj_of(b);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 16 * bi + g + 8 * h;
            const float since = b > 0 ? sm.row[bj][i] : 1.0f, bk = sm.bk[i] * since, rq = sm.rq[i] * since;
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) {
                const int j0 = 16 * bj + 8 * ni + 2 * t;
                float l[2], m[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int j = j0 + e;
                    const float dcy = sm.rk[j] * (b > 0 ? sm.col[j] : j <= i ? expf(float(sm.cum[i] - sm.cum[j])) : 0.0f);
                    l[e] = j < i ? bk * dcy * kk[b][ni][2 * h + e] : 0.0f;
                    m[e] = j <= i ? rq * dcy * qk[b][ni][2 * h + e] : 0.0f;
                }
                // A product with zeros would carry what is no number to rows in front of its own.  It leaves by the row's beta instead:
                // T's column, and with it the walk's U, is none from the row itself on.
                if (!(fabsf(l[0]) + fabsf(l[1]) <= 3.402823466e38f)) {
                    l[0] = l[1] = 0.0f;
                    sm.beta[i] = __int_as_float(0x7fffffff);
                }
                *reinterpret_cast<float2*>(sm.l + i * LP + j0) = make_float2(l[0], l[1]);
                uint32_t mh, ml;
                const int at = tri_step(bj) + (2 * (bi - bj) + h) * 256 + ni * 128 + g * 16 + 4 * t;      // tri_at(i, j0)
                split_pair(m[0], m[1], mh, ml);
                *reinterpret_cast<uint32_t*>(out + W::M + at) = mh;
                *reinterpret_cast<uint32_t*>(out + (LO_WS ? W::ML + at : W::T + sw128(i, j0 >> 3) + 2 * (j0 & 7))) = ml;
            }
        }
    }
    __syncwarp();
    // ---------------------------------------------------------------- X = (I + L)^-1: the blocks on the diagonal by substitution, a column a lane
    if (lane < 16) {
        const float* lrow = sm.l + 16 * warp * (LP + 1);
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s0 = i == lane ? 1.0f : 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const float4 l = *reinterpret_cast<const float4*>(lrow + i * LP + j);
                s0 = fmaf(-l.x, x[j], s0);
                if (j + 1 < i) s1 = fmaf(-l.y, x[j + 1], s1);
                if (j + 2 < i) s2 = fmaf(-l.z, x[j + 2], s2);
                if (j + 3 < i) s3 = fmaf(-l.w, x[j + 3], s3);
            }
            x[i] = (s0 + s1) + (s2 + s3);
            xs[(16 * warp + i) * LP + 16 * warp + lane] = x[i];
        }
    }
    __syncthreads();
    if (!LO_WS)                                                  // M lo to o's rows, a copy in the columns of each CTA of the walk
        for (int v = tid; v < CT * 8; v += 128) {
            const int row = v >> 3, p = v & 7;
            if (row < left && p < 2 * (row >> 4) + 2) {
                const uint4 x = *reinterpret_cast<const uint4*>(out + W::T + sw128(row, p));
                T* o = static_cast<T*>(a.o) + (t0 + row) * a.ldo + head * a.DV + 8 * p;
                for (int c = 0; c < a.DV; c += TV) *reinterpret_cast<uint4*>(o + c) = x;
            }
        }
    // ... then pairs of blocks, X_10 = -X_11 L_10 X_00 and X_32 likewise, then the lower left quarter from the halves on its sides.  A
    // product's result goes through shared memory: over the L that it used up.
    auto L = [&](int i, int j) { return sm.l + 16 * (i * LP + j); };
    auto X = [&](int i, int j) { return xs + 16 * (i * LP + j); };
    if (warp < 2) {
        const int i = 2 * warp + 1, j = 2 * warp;
        float y[2][4] = {}, z[2][4] = {};
        block_product<LP>(y, L(i, j), X(j, j), g, t);
        __syncwarp();
        block_store<LP>(L(i, j), y, 1.0f, g, t);
        __syncwarp();
        block_product<LP>(z, X(i, i), L(i, j), g, t);
        block_store<LP>(X(i, j), z, -1.0f, g, t);
    }
    __syncthreads();
    {
        const int i = 2 + (warp >> 1), j = warp & 1;             // Y = L X of the quarter: Y_i0 = L_i0 X_00 + L_i1 X_10, Y_i1 = L_i1 X_11
        float y[2][4] = {}, z[2][4] = {};
        if (j == 0) block_product<LP>(y, L(i, 0), X(0, 0), g, t);
        block_product<LP>(y, L(i, 1), X(1, j), g, t);
        __syncthreads();                                         // the quarter of L is read
        block_store<LP>(L(i, j), y, 1.0f, g, t);
        __syncthreads();
        if (i == 3) block_product<LP>(z, X(3, 2), L(2, j), g, t);      // X_ij = -(X_i2 Y_2j + X_i3 Y_3j)
        block_product<LP>(z, X(i, i), L(i, j), g, t);
        block_store<LP>(X(i, j), z, -1.0f, g, t);
    }
    __syncthreads();
    {                                                            // T = X diag(beta) in pieces: pairs of columns of the ten blocks, ten a thread
        float2 v[10];
        float top = 0.0f;
#pragma unroll
        for (int b = 0; b < 10; ++b) {
            const int bi = b == 0 ? 0 : b < 3 ? 1 : b < 6 ? 2 : 3, bj = b - bi * (bi + 1) / 2;
            const int i = 16 * bi + (tid >> 3), j = 16 * bj + 2 * (tid & 7);
            const float2 x = *reinterpret_cast<const float2*>(xs + i * LP + j), bt = *reinterpret_cast<const float2*>(sm.beta + j);
            v[b] = make_float2(j > i ? 0.0f : x.x * bt.x, j + 1 > i ? 0.0f : x.y * bt.y);
            top = fmaxf(top, fmaxf(fabsf(v[b].x), fabsf(v[b].y)));
        }
        top = warp_max(top);
        if (lane == 0) sm.top[warp] = top;
        __syncthreads();
        top = fmaxf(fmaxf(sm.top[0], sm.top[1]), fmaxf(sm.top[2], sm.top[3]));
        const int te = clampi(exponent_of(top), 27, 227);
        const float sc = pow2_biased(253 - te);
        if (tid == 0)
            *reinterpret_cast<float4*>(out + W::E64) = make_float4(expf(float(last)), pow2_biased(te + 1), fmaxf(sm.erm[0], sm.erm[1]),
                                                                   pow2_biased(clampi(exponent_of(fmaxf(sm.dkm[0], sm.dkm[1])), 27, 227) + 1));
        const int in_block = (tid >> 6) * 256 + ((tid >> 2) & 1) * 128 + ((tid >> 3) & 7) * 16 + (tid & 3) * 4;
        if (tid < CT) outf(W::DK)[tid] *= pow2_biased(253 - clampi(exponent_of(fmaxf(sm.dkm[0], sm.dkm[1])), 27, 227));
#pragma unroll
        for (int b = 0; b < 10; ++b) {
            const int bi = b == 0 ? 0 : b < 3 ? 1 : b < 6 ? 2 : 3, bj = b - bi * (bi + 1) / 2;
            const int at = tri_step(bj) + (bi - bj) * 512 + in_block;      // tri_at(16 bi + tid / 8, 16 bj + 2 (tid % 8))
            split_pair(v[b].x * sc, v[b].y * sc, *reinterpret_cast<uint32_t*>(out + W::T + at), *reinterpret_cast<uint32_t*>(out + W::TL + at));
        }
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(ws + ((long long)chunk * a.HV + head) * W::BYTES);
    const uint4* src = reinterpret_cast<const uint4*>(out);
    for (int i = tid; i < W::BYTES / 16; i += 128) dst[i] = src[i];
}

// ---------------------------------------------------------------------------------------------------- the walk
// Warps 0-7 the value columns, 8-11 their outputs, 12 the products, 13 the copies, 14 and 15 K and Q to fp16.
constexpr int COMPUTE = 8, OUTPUT = 4, CONVERT = 2, WARP_MMA = 12, WARP_COPY = 13, TC_THREADS = 512;
constexpr uint32_t PREFILL_POLLS = 1u << 17;            // about half a second (4 us a poll)

// A long sequence of few heads is walked in segments of `chunks` chunks side by side.  The state behind a segment is Phi S + X, with S in
// front of it: pass 1 walks every segment but the last from nothing (X), and from the identity without values (Phi); the first one from
// its own state, outputs and all.  gdn_prefill_tc_join_kernel makes X of every segment the state behind it, pass 2 walks the others again
// from there.  Sequence n's segments stand at first_chunk / chunks + n, as its chunks do.
struct WalkSegments {
    int chunks, pass;                                            // 0, 0: no segments
    float* x;                                                    // [place][head][DK][DV]
    float* phi;                                                  // [place][head][column][key]
};
__device__ __forceinline__ int first_segment(int first_chunk, int n, int chunks) { return first_chunk / chunks + n; }
// Place of what a sequence's first segment leaves, the others' behind it.  All but the last leave something, (length - 1) / (64 chunks) of
// them: never over those of n + 1, and no more than n_tokens / (64 chunks) in all.
__device__ __forceinline__ int first_place(const SeqRows& r, int chunks) { return r.start / (CT * chunks); }

// (out of line: the waits' own code has to stay short)
__device__ __noinline__ void give_up(int* abort, int warp) {
    *abort = 1;
    atomicCAS(&g_prefill_status, 0, 1 + (warp < COMPUTE ? 0 : warp < WARP_MMA ? 1 : warp - 10));
}

struct WalkMaps { CUtensorMap q, k, v, o; };                     // 64 rows x 64 columns swizzled, 64 x 128 columns of V as they are

template <int DK, bool LO_WS, int STAGES> struct WalkSmem {
    static constexpr int M_LO = (Ws<LO_WS>::BYTES + 1023) / 1024 * 1024;      // (not LO_WS) M lo from o's rows: 64 of 128 bytes, swizzled
    struct Stage {
        __align__(1024) uint8_t kq[2 * CT * DK * 2];             // scaled fp16 by halves of 64 keys: 64 rows of K, 64 rows of Q, 128 bytes each, swizzled
        __align__(1024) uint8_t v[CT * TV * 2];                  // [token][value] as it is
        __align__(1024) uint8_t w[M_LO + (LO_WS ? 0 : CT * 128)];
    } st[STAGES];
    float vtop[2][TV], meet1[2][TV];                             // the chunk's largest |V| of a column; what its two threads tell each other
    __align__(16) float2 meet2[2][TV];
    __align__(16) float4 scale[TV];                              // and the thread of its outputs: two factors, the first bad token
    __align__(8) uint64_t bars[3 * STAGES + 11];
    uint32_t tmem;
    int abort;
};

// columns of tensor memory
template <int DK> struct Cols {
    static constexpr int P = 0, S = DK, R = 2 * DK, MU = 2 * DK + 64, QS = 2 * DK + 128;     // W lies over P, D over S, U and its pieces over R; two of QS
};

// D[128 x N] (+)= A (tensor memory, fp16) x B (shared memory)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
}
// Waits for a phase of a barrier, at most `polls` times the hardware's own patience; a few instructions, for loops that must stay short.
__device__ __forceinline__ bool mbar_wait_counted(uint32_t bar, uint32_t parity, uint32_t polls) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %3;\n"
        "WAIT_%=:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE_%=;\n\tsub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra WAIT_%=;\n"
        "DONE_%=:\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(polls) : "memory");
    return ok != 0;
}
// (A wait names a phase by its parity: no barrier may get two phases ahead of one that still waits.  Every barrier's next phase follows
// from what its waiters do after the last one, but b_v's, of which there are two.)
//
// the largest magnitude of three; not a number if one is none
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// float32 sums of fp16 products, 128 rows, n columns; the second operand's columns contiguous (`mn`) or its depth
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool mn) { return (1u << 4) | (mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (8u << 24); }
// core matrices of 8 rows x 16 bytes: lbo between the two of a step's depth, sbo between groups of eight rows
__device__ __forceinline__ uint64_t desc_plain(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(lbo >> 4) << 16) | (uint64_t(sbo >> 4) << 32) | (uint64_t(1) << 46);
}
// SWIZZLE_128B, columns contiguous: 64 of them a row of 128 bytes, the next 64 `lbo` further on, eight rows of depth 1,024 bytes
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t lbo) {
    return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(lbo >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void tc_st16(uint32_t t, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t t, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pair_sync(int quad) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory"); }
// registers of a warp group: 512 threads start with 128 each; 2 x 152 + 2 x 104 = 4 x 128
template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int DK, int STAGES>
__global__ void __launch_bounds__(TC_THREADS, 1) gdn_prefill_tc_walk_kernel(const __grid_constant__ WalkMaps maps, const shvk_gdn_seq_args a, const uint8_t* __restrict__ ws, const WalkSegments seg, uint32_t polls, bool starve) {
    constexpr bool LO_WS = M_LO_IN_WS<T>;
    using W = Ws<LO_WS>;
    using Sm = WalkSmem<DK, LO_WS, STAGES>;
    using C = Cols<DK>;
    constexpr int HALF = 2 * CT * 128;                           // bytes of 64 keys of K and Q
    extern __shared__ uint8_t walk_raw[];
    Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(walk_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int splits = (a.DV + TV - 1) / TV, kinds = splits + (seg.pass == 1), split = int(blockIdx.x % unsigned(kinds));
    const int nh = int(blockIdx.x / unsigned(kinds)), head = nh % a.HV, khead = head / (a.HV / a.HK);
    const bool phi = split == splits;                            // this CTA makes the segment's Phi
    const int columns = phi ? DK : min(a.DV - split * TV, TV);   // the lanes behind them walk along, from zero states to nowhere
    int n = nh / a.HV, at = 0, segment = 0;
    if (seg.chunks) {                                            // the last sequence whose first segment is not behind this one
        segment = n;
        n = 0;
        for (int lo = 0, hi = a.n_seq - 1; lo <= hi;) {
            const int mid = (lo + hi) >> 1;
            if (first_segment(first_chunk(SeqRows(a.seq_start, mid, int(a.n_tokens)), mid), mid, seg.chunks) <= segment) { n = mid; lo = mid + 1; } else hi = mid - 1;
        }
    }
    const SeqRows rows(a.seq_start, n, int(a.n_tokens));
    const int all = (rows.end - rows.start + CT - 1) / CT;       // chunks of the sequence; here: NB of them from chunk c0 on
    if (seg.chunks) at = segment - first_segment(first_chunk(rows, n), n, seg.chunks);
    const int c0 = at * seg.chunks, NB = seg.chunks ? min(all - c0, seg.chunks) : all;
    const bool last = c0 + NB >= all;
    next_may_start();
    if (at < 0 || (at > 0 && NB <= 0) ||                         // no segment of any sequence stands here
        (seg.pass == 1 && ((at > 0 && last) || (at == 0 && phi))) || (seg.pass == 2 && at == 0)) {
        last_is_done();
        return;
    }
    const int start = rows.start + c0 * CT, len = rows.end - start;
    const bool writes = seg.pass != 1 || at == 0;                // outputs
    const long long in = at == 0 ? slot_of(a.slot_in, n, a.n_slots) : -1, out = last ? slot_of(a.slot_out, n, a.n_slots) : -1;
    const long long state_of = (long long)a.HV * DK * a.DV, state_at = (long long)head * DK * a.DV + split * TV;
    const int place = seg.chunks ? first_place(rows, seg.chunks) + at : 0;
    // where the state comes from and goes to: columns to_c apart, keys to_k
    const float* from = in >= 0 ? a.states + in * state_of + state_at : seg.pass == 2 ? seg.x + (place - 1) * state_of + state_at : nullptr;
    float* to = last ? (out >= 0 ? a.states + out * state_of + state_at : nullptr) : phi ? seg.phi + ((long long)place * a.HV + head) * DK * DK
                : seg.pass == 1 ? seg.x + place * state_of + state_at : nullptr;
    const long long to_k = phi ? 1 : a.DV, to_c = phi ? DK : 1;
    if (NB <= 0) {                                               // nothing to walk: the state as it is
        last_is_done();
        if (out >= 0 && out != in)
            for (int i = tid; i < DK * TV; i += TC_THREADS) {
                const long long e = (i / TV) * (long long)a.DV + i % TV;
                if (i % TV < columns) to[e] = from ? from[e] : 0.0f;
            }
        return;
    }
    const uint32_t bars = smem_u32(sm.bars);
    auto full = [&](int s) { return bars + 8u * s; };                                    // K and Q of a stage, in fp16
    auto wfull = [&](int s) { return bars + 8u * (STAGES + s); };                        // all of it, as it is
    auto empty = [&](int s) { return bars + 8u * (2 * STAGES + s); };
    const uint32_t b_s = bars + 8u * (3 * STAGES), b_r = b_s + 8, b_w = b_s + 16, b_u = b_s + 24, b_d = b_s + 32, b_p = b_s + 40, b_o = b_s + 48, b_q = b_s + 56,
                   b_m = b_s + 64, b_v = b_s + 72;
    if (tid == 0) {
        sm.abort = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 32 * CONVERT);
            mbar_init(wfull(s), 1);
            mbar_init(empty(s), COMPUTE + OUTPUT + 1);
        }
        mbar_init(b_s, COMPUTE); mbar_init(b_w, COMPUTE); mbar_init(b_d, COMPUTE); mbar_init(b_q, OUTPUT); mbar_init(b_v, OUTPUT); mbar_init(b_v + 8, OUTPUT); mbar_init(b_m, COMPUTE / 2);
        mbar_init(b_r, 1); mbar_init(b_u, 1); mbar_init(b_p, 1); mbar_init(b_o, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == WARP_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    last_is_done();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;                               // 0: the columns are all there are
    // A role whose wait has given up goes on through its loop without waiting, issuing or writing, so that the barriers among warps are
    // met by all; those that wait for it give up in turn.
    bool dead = tmem != 0;
    if (dead && tid == 0) atomicCAS(&g_prefill_status, 0, 8);
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (__any_sync(0xffffffffu, !mbar_wait_counted(bar, parity & 1u, polls))) {
            dead = true;
            polls = 1;
            give_up(&sm.abort, warp);
        }
    };
    constexpr float FINITE = 3.402823466e38f;

    if (warp < COMPUTE) {
        // ------------------------------------------------------------------------------------------- the value columns
        regs_up<152>();
        constexpr int KH = DK / 2;                               // keys of a thread
        const int quad = warp & 3, half = warp >> 2, row = 32 * quad + lane;
        const uint32_t tl = uint32_t(32 * quad) << 16;
        float S[KH], sig = 1.0f, inv = 1.0f, mine = 0.0f;       // S in units of inv; mine: the largest |S| here
        {
            const float* src = from + (long long)(half * KH) * a.DV + row;
#pragma unroll
            for (int i = 0; i < KH; ++i) {
                S[i] = from && row < columns ? src[i * (long long)a.DV] : phi && row == half * KH + i ? 1.0f : 0.0f;
                mine = fmaxf(mine, fabsf(S[i]));
            }
            sm.meet1[half][row] = mine;
            pair_sync(quad);
            const float m = fmaxf(mine, sm.meet1[half ^ 1][row]);
            const int b = m > 0.0f ? clampi(265 - exponent_of(m), 27, 191) : 127;        // m sig in [2^11, 2^12)
            sig = pow2_biased(b);
            inv = pow2_biased(254 - b);
#pragma unroll
            for (int i = 0; i < KH; ++i) S[i] *= sig;
            mine *= sig;
            pair_sync(quad);                                     // meet1 is read
        }
        int s = 0;
        uint32_t sph = 0;
#pragma unroll 1
        for (int c = 0; c < NB; ++c) {
            const typename Sm::Stage& st = sm.st[s];
            const uint32_t ph = uint32_t(c) & 1u;
            const float* sc = reinterpret_cast<const float*>(st.w);
            // ------------------------------------------------------------------- pieces of S
#pragma unroll
            for (int p = 0; p < KH / 32; ++p) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) split_pair(S[32 * p + 2 * i], S[32 * p + 2 * i + 1], hi[i], lo[i]);
                tc_st16(tl + C::S + half * (KH / 2) + 16 * p, hi);
                tc_st16(tl + C::S + DK / 2 + half * (KH / 2) + 16 * p, lo);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_s);
            // What is no number, or none any more, belongs to its own token and those behind it.  It leaves the products, whose zeros would
            // carry it to tokens in front of it; the column's outputs from there on, and its state, are marked instead.
            int first = CT;
            auto clean = [&](float (&x)[16], int p) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i += 2) m = max3_nan(m, x[i], x[i + 1]);
                if (!(m <= FINITE))
#pragma unroll
                    for (int i = 15; i >= 0; --i)
                        if (!(fabsf(x[i]) <= FINITE)) {
                            first = min(first, 32 * half + 16 * p + i);
                            x[i] = 0.0f;
                        }
            };
            // ------------------------------------------------------------------- while K S0 runs: a bound of W
            wait(wfull(s), sph);
            wait(full(s), sph);                                  // (V's rows past the sequence are cleared with K and Q)
            wait(b_v + 8 * ph, uint32_t(c >> 1));
            const T* v = reinterpret_cast<const T*>(st.v) + 32 * half * TV + row;
            sm.meet1[half][row] = mine;
            pair_sync(quad);
            const float vtop = sm.vtop[ph][row], stop = fmaxf(mine, sm.meet1[half ^ 1][row]);      // stop: the column's largest |S|
            const float4 tail = *reinterpret_cast<const float4*>(st.w + W::E64);     // e_64, T's scale, the largest ER, DK's scale
            const float e64 = tail.x;
            // |W| <= |V| + max ER |K'| |S|, |K'| < 1: at most 2^8 in its scale, so that U, a sum of 64, is within 2^14
            // (not below 2^-55: the product of two scales, sig up to 2^64, has to stay finite)
            const int wb = clampi(exponent_of(fmaf(vtop, sig, tail.z * stop * (DK == 64 ? 8.0f : 11.4f))), 72, 227);
            const float wsc = pow2_biased(261 - wb), uf = pow2_biased(wb - 7) * tail.y;
            float scaled[32];                                    // V in W's scale
#pragma unroll
            for (int i = 0; i < 32; ++i) scaled[i] = to_float(v[i * TV]) * (sig * wsc);
            wait(b_r, ph);
            tc_fence_after();
            // ------------------------------------------------------------------- W = V - e K S0
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                uint32_t r[16], hi[8], lo[8];
                tc_ld16(tl + C::R + 32 * half + 16 * p, r);
                float (&x)[16] = *reinterpret_cast<float (*)[16]>(scaled + 16 * p);
                const float2 ws2 = make_float2(-wsc, -wsc);
                const float4* er4 = reinterpret_cast<const float4*>(sc + W::ER / 4 + 32 * half + 16 * p);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 er = er4[i / 4];
                    const float2 a0 = fma2(mul2(make_float2(er.x, er.y), ws2), make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), make_float2(x[i], x[i + 1]));
                    const float2 a1 = fma2(mul2(make_float2(er.z, er.w), ws2), make_float2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])), make_float2(x[i + 2], x[i + 3]));
                    x[i] = a0.x; x[i + 1] = a0.y; x[i + 2] = a1.x; x[i + 3] = a1.y;
                }
                clean(x, p);
#pragma unroll
                for (int i = 0; i < 8; ++i) split_pair(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
                tc_st8(tl + C::P + 16 * half + 8 * p, hi);
                tc_st8(tl + C::P + 32 + 16 * half + 8 * p, lo);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_w);
            wait(b_u, ph);
            tc_fence_after();
            // ------------------------------------------------------------------- pieces of U, and of D = exp(c_64 - c_j) U
            float sum = 0.0f, f = 1.0f;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                float x[16];
                uint32_t hi[8], lo[8];
                tc_ld16(tl + C::R + 32 * half + 16 * p, reinterpret_cast<uint32_t*>(x));
                const float4* dk4 = reinterpret_cast<const float4*>(sc + W::DK / 4 + 32 * half + 16 * p);
                tc_wait_ld();
                clean(x, p);
#pragma unroll
                for (int i = 0; i < 8; ++i) split_pair(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
                tc_st8(tl + C::R + 32 * half + 16 * p, hi);      // over the U that this round has read
                tc_st8(tl + C::R + 32 * half + 16 * p + 8, lo);
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 dk = dk4[i / 4];
                    const float2 d0 = mul2(make_float2(x[i], x[i + 1]), make_float2(dk.x, dk.y)), d1 = mul2(make_float2(x[i + 2], x[i + 3]), make_float2(dk.z, dk.w));
                    sum += (fabsf(d0.x) + fabsf(d0.y)) + (fabsf(d1.x) + fabsf(d1.y));
                    split_pair(d0.x, d0.y, hi[i / 2], lo[i / 2]);
                    split_pair(d1.x, d1.y, hi[i / 2 + 1], lo[i / 2 + 1]);
                }
                tc_st8(tl + C::S + 16 * half + 8 * p, hi);
                tc_st8(tl + C::S + 32 + 16 * half + 8 * p, lo);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_d);
            // ------------------------------------------------------------------- while K^T D runs: a bound of the new state, its scale
            sm.meet2[half][row] = make_float2(sum, __int_as_float(first));
            pair_sync(quad);
            const float du = uf * tail.w;                        // of a unit of K^T D in the state's
            {
                const float2 o2 = sm.meet2[half ^ 1][row];
                first = min(first, __float_as_int(o2.y));
                const float top = fmaf(e64, stop, du * (sum + o2.x));      // |k| < 1 in its units
                if (!(top <= 32768.0f && (top >= 512.0f || top == 0.0f))) {
                    const int b = exponent_of(sig);
                    const int nb = top > 0.0f ? clampi(b + clampi(138 - exponent_of(top), -100, 100), 27, 191) : b;     // top f in [2^11, 2^12)
                    f = pow2_biased(127 + clampi(nb - b, -120, 120));
                }
            }
            wait(b_q, ph ^ 1u);                       // the last chunk's outputs have read theirs
            if (half == 0) sm.scale[row] = make_float4(inv, inv * uf, __int_as_float(first), 0.0f);
            __syncwarp();
            if (lane == 0) {
                if (half == 0) mbar_arrive(b_m);
                mbar_arrive(empty(s));
            }
            const float ef = e64 * f, df = first < CT ? __int_as_float(0x7fffffff) : du * f;
            wait(b_p, ph);
            tc_fence_after();
            // ------------------------------------------------------------------- S = e_64 S0 + K^T D
            mine = 0.0f;
            {
                uint32_t r[KH];
#pragma unroll
                for (int p = 0; p < KH / 32; ++p) tc_ld32(tl + C::P + half * KH + 32 * p, r + 32 * p);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < KH; i += 2) {
                    const float2 u = mul2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), make_float2(df, df));
                    const float2 w = fma2(make_float2(ef, ef), make_float2(S[i], S[i + 1]), u);
                    S[i] = w.x;
                    S[i + 1] = w.y;
                    mine = max3_nan(mine, w.x, w.y);
                }
            }
            sig *= f;
            inv = pow2_biased(254 - exponent_of(sig));
            if (++s == STAGES) { s = 0; sph ^= 1u; }
        }
        if (to && !dead && row < columns) {
            float* dst = to + (half * KH) * to_k + row * to_c;
#pragma unroll
            for (int i = 0; i < KH; ++i) dst[i * to_k] = S[i] * inv;
        }
    } else if (warp < COMPUTE + OUTPUT) {
        // ------------------------------------------------------------------------------------------- O = M U + e Q S0
        regs_down<104>();
        const int quad = warp & 3, row = 32 * quad + lane;
        const uint32_t tl = uint32_t(32 * quad) << 16;
        T* o = static_cast<T*>(a.o) + start * a.ldo + (long long)head * a.DV + split * TV + row;
        int s = 0, sn = 0;                                       // stages of the chunk to write and of the next one
        uint32_t sph = 0, snph = 0;
        auto next_top = [&](int c) {                             // the largest |V| of chunk c: what W will be scaled by (an infinity sets no scale)
            if (c >= NB) return;
            wait(wfull(sn), snph);
            wait(full(sn), snph);
            const T* v = reinterpret_cast<const T*>(sm.st[sn].v) + row;
            float m = 0.0f;
#pragma unroll 1
            for (int p = 0; p < CT; p += 16)
#pragma unroll
                for (int i = 0; i < 16; i += 2) m = max3_nan(m, to_float(v[(p + i) * TV]), to_float(v[(p + i + 1) * TV]));
            if (!(m <= FINITE)) {
                m = 0.0f;
#pragma unroll 1
                for (int p = 0; p < CT; ++p) {
                    const float y = fabsf(to_float(v[p * TV]));
                    m = y <= FINITE ? fmaxf(m, y) : m;
                }
            }
            sm.vtop[c & 1][row] = m;
            __syncwarp();
            if (lane == 0) mbar_arrive(b_v + 8 * (c & 1));     // (two barriers: this may be a chunk ahead of those that wait)
            if (++sn == STAGES) { sn = 0; snph ^= 1u; }
        };
        next_top(0);
#pragma unroll 1
        for (int c = 0; c < NB; ++c) {
            const typename Sm::Stage& st = sm.st[s];
            const uint32_t ph = uint32_t(c) & 1u;
            const float* sc = reinterpret_cast<const float*>(st.w);
            next_top(c + 1);
            wait(b_m, ph);
            wait(b_o, ph);
            tc_fence_after();
            const float4 mark = sm.scale[row];
            const int first = __float_as_int(mark.z), left = dead || !writes || 32 * quad >= columns ? 0 : len - c * CT;     // (columns: 64 or 128)
            const bool plain = __all_sync(0xffffffffu, left >= CT && first >= CT);
            // sixteen tokens at a time in a loop: the code of a chunk's roles has to fit the instruction cache
#pragma unroll 1
            for (int h = left > 0 ? 0 : 3; h < 4; ++h) {         // (without outputs: the last round, for its barrier)
                uint32_t q[16], m[16];
                tc_ld16(tl + C::QS + 64 * ph + 16 * h, q);
                tc_ld16(tl + C::MU + 16 * h, m);
                tc_wait_ld();
                if (h == 3) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b_q);
                }
                if (left <= 0) break;
                T* at = o + 16 * h * a.ldo;
                const float4* om4 = reinterpret_cast<const float4*>(sc + W::OM / 4 + 16 * h);
                const float4* eq4 = reinterpret_cast<const float4*>(sc + W::EQ / 4 + 16 * h);
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 om = om4[i / 4], eq = eq4[i / 4];
                    const float2 a0 = mul2(mul2(make_float2(om.x, om.y), make_float2(mark.y, mark.y)), make_float2(__uint_as_float(m[i]), __uint_as_float(m[i + 1])));
                    const float2 a1 = mul2(mul2(make_float2(om.z, om.w), make_float2(mark.y, mark.y)), make_float2(__uint_as_float(m[i + 2]), __uint_as_float(m[i + 3])));
                    const float2 x0 = fma2(mul2(make_float2(eq.x, eq.y), make_float2(mark.x, mark.x)), make_float2(__uint_as_float(q[i]), __uint_as_float(q[i + 1])), a0);
                    const float2 x1 = fma2(mul2(make_float2(eq.z, eq.w), make_float2(mark.x, mark.x)), make_float2(__uint_as_float(q[i + 2]), __uint_as_float(q[i + 3])), a1);
                    m[i / 2] = pack2<T>(x0.x, x0.y);
                    m[i / 2 + 1] = pack2<T>(x1.x, x1.y);
                }
                const T* two = reinterpret_cast<const T*>(m);
                if (plain) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        *at = two[i];
                        at += a.ldo;
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < 16; ++i) {               // (few chunks: the last of a sequence, or one with a bad token)
                        const uint32_t word = i < 8 ? (i < 4 ? (i < 2 ? m[0] : m[1]) : (i < 6 ? m[2] : m[3])) : (i < 12 ? (i < 10 ? m[4] : m[5]) : (i < 14 ? m[6] : m[7]));
                        const T x = reinterpret_cast<const T*>(&word)[i & 1];
                        if (16 * h + i < left) *at = 16 * h + i < first ? x : from_float<T>(__int_as_float(0x7fffffff));
                        at += a.ldo;
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(s));
            o += CT * a.ldo;
            if (++s == STAGES) { s = 0; sph ^= 1u; }
        }
    } else {
        regs_down<104>();
        if (warp == WARP_MMA) {
            // --------------------------------------------------------------------------------------- the products
            const bool lead = elect_one();
            // (in loops: unrolled, the products of a chunk take 13 KB of code, for which the other roles' leaves the instruction cache: 8 % slower)
            auto products = [&](int c, int s, uint32_t sph) {
                const uint32_t ph = uint32_t(c) & 1u;
                const uint32_t kq = smem_u32(sm.st[s].kq), wt = smem_u32(sm.st[s].w);
                constexpr uint32_t id64 = idesc_f16(64, false);
                wait(full(s), sph);
                wait(b_o, ph ^ 1u);                              // M U has read the pieces of U, which K S0 overwrites
                wait(b_s, ph);
                tc_fence_after();
                const uint32_t qs = C::QS + 64 * ph;             // (read by the outputs of chunk c - 2 before M U of chunk c - 1 was let in)
                if (!dead && lead) {
                    const uint64_t b0 = smem_desc_sw128(kq);
#pragma unroll 1
                    for (int p = 0; p < DK / 16; ++p) {          // (K S0)^T, for which the chain waits
                        const uint64_t b = b0 + uint64_t((p >> 2) * (HALF / 16) + 2 * (p & 3));
                        mma_ts(C::R, C::S + 8 * p, b, id64, p > 0);
                        mma_ts(C::R, C::S + DK / 2 + 8 * p, b, id64, true);
                    }
                    tc_commit(b_r);
#pragma unroll 1
                    for (int p = 0; p < DK / 16; ++p) {          // (Q S0)^T
                        const uint64_t b = b0 + uint64_t((p >> 2) * (HALF / 16) + 2 * (p & 3) + CT * 128 / 16);
                        mma_ts(qs, C::S + 8 * p, b, id64, p > 0);
                        mma_ts(qs, C::S + DK / 2 + 8 * p, b, id64, true);
                    }
                }
                wait(wfull(s), sph);
                wait(b_w, ph);
                tc_fence_after();
                if (!dead && lead) {
                    const uint64_t t0 = desc_plain(wt, 128, 256);
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) {             // T is triangular: tokens 16 kk .. reach columns 16 kk .. 63
                        const uint64_t th = t0 + uint64_t((W::T + tri_step(kk)) / 16), tlo = t0 + uint64_t((W::TL + tri_step(kk)) / 16);
                        const uint32_t id = idesc_f16(64 - 16 * kk, false), d = C::R + 16 * kk;
                        mma_ts(d, C::P + 8 * kk, th, id, kk > 0);
                        mma_ts(d, C::P + 8 * kk, tlo, id, true);
                        mma_ts(d, C::P + 32 + 8 * kk, th, id, true);
                    }
                    tc_commit(b_u);
                }
                wait(b_d, ph);
                tc_fence_after();
                if (!dead && lead) {
                    constexpr uint32_t idk = idesc_f16(DK, true);
                    const uint64_t b0 = desc_mn(kq, HALF);
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) {
                        mma_ts(C::P, C::S + 8 * kk, b0 + uint64_t(128 * kk), idk, kk > 0);
                        mma_ts(C::P, C::S + 32 + 8 * kk, b0 + uint64_t(128 * kk), idk, true);
                    }
                    tc_commit(b_p);
                }
                wait(b_q, ph ^ 1u);                   // the last chunk's outputs are read
                tc_fence_after();
                if (!dead && lead) {
                    const uint64_t m0 = desc_plain(wt, 128, 256), o0 = smem_desc_sw128(wt + Sm::M_LO);
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t mh = m0 + uint64_t((W::M + tri_step(kk)) / 16);
                        const uint32_t id = idesc_f16(64 - 16 * kk, false), d = C::MU + 16 * kk, u = C::R + 16 * kk;
                        mma_ts(d, u, mh, id, kk > 0);
                        mma_ts(d, u, LO_WS ? m0 + uint64_t((W::ML + tri_step(kk)) / 16) : o0 + uint64_t(kk * (16 * 128 / 16 + 2)), id, true);
                        mma_ts(d, u + 8, mh, id, true);
                    }
                    tc_commit(b_o);
                    tc_commit(empty(s));
                }
            };
            int s = 0;
            uint32_t sph = 0;
#pragma unroll 1
            for (int c = 0; c < NB; ++c) {
                products(c, s, sph);
                if (++s == STAGES) { s = 0; sph ^= 1u; }
            }
        } else if (warp == WARP_COPY) {
            // --------------------------------------------------------------------------------------- copies
            const uint8_t* src = ws + ((long long)(first_chunk(rows, n) + c0) * a.HV + head) * W::BYTES;
            const uint32_t lead = elect_one();
            int s = 0;
            uint32_t sph = 0;
#pragma unroll 1
            for (int c = 0; c < NB; ++c) {
                const uint32_t kq = smem_u32(sm.st[s].kq), vt = smem_u32(sm.st[s].v), wt = smem_u32(sm.st[s].w);
                const int y = start + c * CT;
                wait(empty(s), sph ^ 1u);
                if (!dead && lead && !(starve && c == 0)) {      // rows past the sequence are another's, past the last zeros: both unused
                    mbar_expect_tx(wfull(s), W::BYTES + 2 * CT * DK * 2 + CT * TV * 2 + (LO_WS ? 0 : CT * 128));
#pragma unroll
                    for (int h = 0; h < DK / 64; ++h) {
                        tma_load_2d(kq + h * HALF, &maps.k, khead * DK + 64 * h, y, wfull(s));
                        tma_load_2d(kq + h * HALF + CT * 128, &maps.q, khead * DK + 64 * h, y, wfull(s));
                    }
                    tma::load_bulk(wt, src + (long long)c * a.HV * W::BYTES, W::BYTES, wfull(s));
                    tma_load_2d(vt, &maps.v, head * a.DV + (phi ? 0 : split * TV), y, wfull(s));
                    if (!LO_WS) tma_load_2d(wt + Sm::M_LO, &maps.o, head * a.DV + (phi ? 0 : split * TV), y, wfull(s));
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; sph ^= 1u; }
            }
        } else {
            // --------------------------------------------------------------------------------------- K and Q to fp16
            // turned in place, eight pieces of 16 bytes at a time: a thread has the same piece of every STEP-th row
            constexpr int NT = 32 * CONVERT, ROWP = DK / 8, STEP = NT / ROWP, PIECES = CT / STEP;
            const int lt = tid - 32 * (WARP_COPY + 1), p = lt % ROWP, r0 = lt / ROWP;
            auto turn = [&](uint4 x, float f) {
                uint32_t* e = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const T* two = reinterpret_cast<const T*>(&e[u]);
                    const float2 v = mul2(make_float2(to_float(two[0]), to_float(two[1])), make_float2(f, f));
                    e[u] = pack_half(v.x, v.y);
                }
                return x;
            };
            int s = 0;
            uint32_t sph = 0;
#pragma unroll 1
            for (int c = 0; c < NB; ++c) {
                typename Sm::Stage& st = sm.st[s];
                const int left = len - c * CT;
                wait(wfull(s), sph);
                const float* ks = reinterpret_cast<const float*>(st.w + W::KS) + r0;
                const float* qs = reinterpret_cast<const float*>(st.w + W::QS) + r0;
                uint8_t* base = st.kq + (p >> 3) * HALF;
#pragma unroll 1
                for (int b = 0; b < PIECES; b += 4) {
                    uint4 k[4], q[4];
                    uint4* at[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        at[i] = reinterpret_cast<uint4*>(base + sw128(r0 + (b + i) * STEP, p & 7));
                        k[i] = *at[i];
                        q[i] = at[i][CT * 128 / 16];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool has = r0 + (b + i) * STEP < left;
                        const uint4 z = make_uint4(0, 0, 0, 0);
                        *at[i] = has ? turn(k[i], ks[(b + i) * STEP]) : z;
                        at[i][CT * 128 / 16] = has ? turn(q[i], qs[(b + i) * STEP]) : z;
                    }
                }
                if (left < CT || phi)                            // (Phi has no values)
                    for (int i = (phi ? 0 : left * (TV / 8)) + lt; i < CT * (TV / 8); i += NT) reinterpret_cast<uint4*>(st.v)[i] = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
                mbar_arrive(full(s));
                if (++s == STAGES) { s = 0; sph ^= 1u; }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (sm.abort) {                                               // products may still be on their way: a millisecond is a thousand times theirs
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    tc_fence_after();
    if (warp == WARP_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// X of segment g becomes Phi_g X_(g-1) + X_g, g = 1 .. the last but one, in float32: a CTA takes JC columns of a head through all segments
// of a sequence, the state so far in shared memory.  A thread has one key of the result and a share of the sum's keys; its part of the
// next Phi does not depend on the state and is on its way while this one is used.  (A segment's Phi, 64 KB out of L2, its products, two
// barriers and a sum are a chain of about 2.3 us; with a whole sum in each thread it took three times that.)
constexpr int JC = 8, JOIN_THREADS = 512;
template <int DK> __global__ void __launch_bounds__(JOIN_THREADS) gdn_prefill_tc_join_kernel(const shvk_gdn_seq_args a, const WalkSegments seg) {
    constexpr int SHARES = JOIN_THREADS / DK, KPT = DK / SHARES, EPT = DK * JC / JOIN_THREADS;      // EPT: values of the result a thread adds up
    static_assert(JC % EPT == 0, "a thread's values lie side by side");
    __shared__ __align__(16) float s[DK][JC], part[SHARES][DK][JC + 1];
    const int parts = a.DV / JC, block = int(blockIdx.x % unsigned(parts)), nh = int(blockIdx.x / unsigned(parts)), n = nh / a.HV, head = nh % a.HV;
    const SeqRows rows(a.seq_start, n, int(a.n_tokens));
    const int segments = ((rows.end - rows.start + CT - 1) / CT + seg.chunks - 1) / seg.chunks;
    next_may_start();
    last_is_done();
    if (segments < 3) return;
    const int key = threadIdx.x % DK, share = threadIdx.x / DK;
    const int k1 = threadIdx.x * EPT / JC, c1 = threadIdx.x * EPT % JC;
    const long long first = first_place(rows, seg.chunks), state_of = (long long)a.HV * DK * a.DV, phi_of = (long long)a.HV * DK * DK;
    float* x = seg.x + first * state_of + ((long long)head * DK + k1) * a.DV + block * JC + c1;
    const float* phi = seg.phi + (first * a.HV + head) * DK * DK + (long long)(share * KPT) * DK + key;
    float p[KPT], y[EPT];
    auto fetch = [&](int g) {
#pragma unroll
        for (int k = 0; k < KPT; ++k) p[k] = phi[g * phi_of + k * DK];
#pragma unroll
        for (int u = 0; u < EPT; ++u) y[u] = x[g * state_of + u];
    };
#pragma unroll
    for (int u = 0; u < EPT; ++u) s[k1][c1 + u] = x[u];
    fetch(1);
    for (int g = 1; g < segments - 1; ++g) {
        float acc[JC] = {};
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
            const float4 lo = *reinterpret_cast<const float4*>(&s[share * KPT + k][0]), hi = *reinterpret_cast<const float4*>(&s[share * KPT + k][4]);
            acc[0] = fmaf(p[k], lo.x, acc[0]); acc[1] = fmaf(p[k], lo.y, acc[1]); acc[2] = fmaf(p[k], lo.z, acc[2]); acc[3] = fmaf(p[k], lo.w, acc[3]);
            acc[4] = fmaf(p[k], hi.x, acc[4]); acc[5] = fmaf(p[k], hi.y, acc[5]); acc[6] = fmaf(p[k], hi.z, acc[6]); acc[7] = fmaf(p[k], hi.w, acc[7]);
        }
        float sum[EPT];
#pragma unroll
        for (int u = 0; u < EPT; ++u) sum[u] = y[u];
        if (g + 1 < segments - 1) fetch(g + 1);
#pragma unroll
        for (int c = 0; c < JC; ++c) part[share][key][c] = acc[c];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < EPT; ++u) {
#pragma unroll
            for (int h = 0; h < SHARES; ++h) sum[u] += part[h][k1][c1 + u];
            s[k1][c1 + u] = sum[u];
            x[g * state_of + u] = sum[u];
        }
    }
}

// Chunks of a segment, 0 where sequences are walked whole.  Counted in chunks' times of one wave of CTAs (a walk's chunk takes 3.8 us, a
// join's segment 2.3, the two launches more about as much as two chunks) for sequences of the average length; segments are not
// shorter than 13 chunks, so that their states take less room than their chunks' T and M.  us, 6 heads of 128 x 128, in segments / whole: 1
// sequence of 2,600 141 / 174, of 16,384 242 / 996; 4 of 3,000 184 / 216; 8 of 4,000 290 / 317; 16 of 8,000, which stay whole, 725.  What
// a join's segment is counted as hardly matters: at 0.15 chunks 1 of 16,384 241, 8 of 4,000 288, but one head of 50,000 275 instead of 271.
inline int segment_chunks(const shvk_gdn_seq_args& a) {
    const long long sms = device_sms(), splits = (a.DV + TV - 1) / TV, heads = (long long)a.n_seq * a.HV, chunks = a.n_tokens / CT / a.n_seq;
    auto waves = [&](long long ctas) { return (ctas + sms - 1) / sms; };
    double best = 0.9 * double(chunks * waves(heads * splits));
    int found = 0;
    for (long long g = 2; g <= 64 && (chunks + g - 1) / g >= 13; ++g) {
        const long long len = (chunks + g - 1) / g;
        const double t = double(len * (waves(heads * (splits + (g - 2) * (splits + 1))) + waves(heads * splits * (g - 1)))) + 0.6 * double(g - 2) + 2.0;
        if (t < best) { best = t; found = int(len); }
    }
    return found;
}
inline long long segment_count(const shvk_gdn_seq_args& a, int chunks) { return (a.n_tokens / CT + a.n_seq + 1) / chunks + a.n_seq + 1; }
inline long long place_count(const shvk_gdn_seq_args& a, int chunks) { return a.n_tokens / (CT * (long long)chunks); }
// The last sequence's chunks end at start / 64 + n_seq - 1 + ceil(length / 64), no more than this.
inline long long chunk_count(const shvk_gdn_seq_args& a) { return a.n_tokens / CT + a.n_seq; }
inline size_t chunk_bytes(const shvk_gdn_seq_args& a) {
    return size_t(chunk_count(a)) * size_t(a.HV) * (a.dtype == DT_F16 ? Ws<true>::BYTES : Ws<false>::BYTES);
}

template <typename T, int DK> int launch_tc(const shvk_gdn_seq_args& a, uint8_t* ws, cudaStream_t s, uint32_t polls, bool starve) {
    constexpr bool LO_WS = M_LO_IN_WS<T>;
    constexpr int STAGES = 3;
    const int chunks = segment_chunks(a);
    const long long segments = chunks ? segment_count(a, chunks) : 0, splits = (a.DV + TV - 1) / TV;
    const long long items = chunk_count(a) * a.HV, ctas = (chunks ? segments : a.n_seq) * a.HV * (splits + (chunks ? 1 : 0));
    if (items > 0x7fffffff || ctas > 0x7fffffff) return int(cudaErrorInvalidValue);
    constexpr int prep_smem = int(sizeof(PrepSmem<DK, LO_WS>)) + 1024, smem = int(sizeof(WalkSmem<DK, LO_WS, STAGES>)) + 1024;
    static_assert(smem <= 227 * 1024, "the stages fit");
    cudaError_t e = cudaFuncSetAttribute(gdn_prefill_tc_prep_kernel<T, DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, prep_smem);
    if (e != cudaSuccess) return int(e);
    e = cudaFuncSetAttribute(gdn_prefill_tc_walk_kernel<T, DK, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return int(e);
    WalkMaps maps;
    if (!tma::make_map_2d(&maps.q, a.q, 2, a.n_tokens, (long long)a.HK * DK, a.ldq, CT, 64, true) ||
        !tma::make_map_2d(&maps.k, a.k, 2, a.n_tokens, (long long)a.HK * DK, a.ldk, CT, 64, true) ||
        !tma::make_map_2d(&maps.v, a.v, 2, a.n_tokens, (long long)a.HV * a.DV, a.ldv, CT, TV, false) ||
        !tma::make_map_2d(&maps.o, a.o, 2, a.n_tokens, (long long)a.HV * a.DV, a.ldo, CT, 64, true))
        return int(cudaErrorInvalidValue);
    // Ahead of the end of what ran before, but for calls in segments: calls in a row of 321 tokens 36.1 -> 34.0 us, of 64 x 2,048 tokens
    // 615.6 -> 614.6, but in segments 1 x 16,384 233.7 -> 235.2.
    if (!chunks) {
        e = launch_behind(gdn_prefill_tc_prep_kernel<T, DK>, items, 128, prep_smem, s, a, ws);
    } else {
        gdn_prefill_tc_prep_kernel<T, DK><<<unsigned(items), 128, prep_smem, s>>>(a, ws);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return int(e);
    WalkSegments seg{};
    auto walk = [&](long long n) { return launch_behind(gdn_prefill_tc_walk_kernel<T, DK, STAGES>, n, TC_THREADS, smem, s, maps, a, ws, seg, polls, starve); };
    if (!chunks) return int(walk(ctas));
    seg.chunks = chunks;
    seg.x = reinterpret_cast<float*>(ws + chunk_bytes(a));
    seg.phi = seg.x + place_count(a, chunks) * a.HV * DK * a.DV;
    seg.pass = 1;
    if ((e = walk(ctas)) != cudaSuccess) return int(e);
    if ((e = launch_behind(gdn_prefill_tc_join_kernel<DK>, (long long)a.n_seq * a.HV * (a.DV / JC), JOIN_THREADS, 0, s, a, seg)) != cudaSuccess) return int(e);
    seg.pass = 2;
    return int(walk(segments * a.HV * splits));
}

}  // namespace

size_t gdn_prefill_tc_workspace(const shvk_gdn_seq_args& a) {
    const int chunks = segment_chunks(a);
    return chunk_bytes(a) + (chunks ? size_t(place_count(a, chunks)) * size_t(a.HV) * size_t(a.DK) * size_t(a.DK + a.DV) * sizeof(float) : 0);
}
int gdn_prefill_tc(const shvk_gdn_seq_args& a, uint8_t* ws, cudaStream_t s, int starve_polls) {
    const bool starve = starve_polls > 0;
    const uint32_t polls = starve ? uint32_t(starve_polls < 256 ? 256 : starve_polls > (1 << 17) ? 1 << 17 : starve_polls) : PREFILL_POLLS;
    if (a.dtype == DT_BF16) return a.DK == 64 ? launch_tc<__nv_bfloat16, 64>(a, ws, s, polls, starve) : launch_tc<__nv_bfloat16, 128>(a, ws, s, polls, starve);
    return a.DK == 64 ? launch_tc<__half, 64>(a, ws, s, polls, starve) : launch_tc<__half, 128>(a, ws, s, polls, starve);
}

}  // namespace sb

extern "C" int shvk_gdn_prefill_status(int* status_out) {
    if (!status_out) return int(cudaErrorInvalidValue);
    return int(cudaMemcpyFromSymbol(status_out, sb::g_prefill_status, sizeof(int)));
}

extern "C" int shvk_gdn_prefill_status_fetch_async(int* host_word, void* stream) {
    if (!host_word) return int(cudaErrorInvalidValue);
    return int(cudaMemcpyFromSymbolAsync(host_word, sb::g_prefill_status, sizeof(int), 0, cudaMemcpyDeviceToHost, cudaStream_t(stream)));
}

extern "C" int shvk_gdn_prefill_status_clear_async(void* stream) {
    void* word = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&word, sb::g_prefill_status);
    return int(e != cudaSuccess ? e : cudaMemsetAsync(word, 0, sizeof(int), cudaStream_t(stream)));
}
