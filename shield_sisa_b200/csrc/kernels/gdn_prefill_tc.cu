// The chunked delta rule with kept states for heads of 128 values (or a multiple): chunks of 64 tokens on tcgen05.  The algebra, the
// pieces and the scales are those of gdn_prefill.cu, with 64 for 16:
//
//     U = T (V - diag(e) K S0),  O = M U + diag(e) Q S0,  S = e_64 S0 + K^T diag(exp(c_64 - c_j)) U
//
// prep   a CTA per chunk and head: T and M, what needs no state.  Gram products of 16 x 16 blocks on mma.sync, the 64 x 64 triangular
//        inverse by block columns in float32, one a warp.  Both leave as fp16 pieces in the layout that the tensor core reads, the
//        blocks above the diagonal left out: 16,912 bytes a chunk (22,032 with the second piece of M).
// walk   a CTA per head and 128 value columns.  The values are the 128 lanes of tensor memory: S^T, W^T, U^T and D^T are operands that
//        lie there as pieces, K, Q, T and M come from shared memory.  The state itself stays in registers: a value column's keys in two
//        threads (eight warps), rounded by float32 FMAs; per chunk its pieces go to tensor memory and the product K^T D comes back.
//        One warp issues the products; three bring K and Q (scaled and turned into fp16 on the way), V, T and M, a chunk or two ahead.
//
// A chunk is a chain: pieces of S -> K S0 -> W -> T W -> D -> K^T D -> S.  Q S0 and M U run beside it, and the outputs of a chunk are
// written while the next one's first product runs.
#include "gdn_pieces.cuh"
#include "gdn_seq.cuh"
#include "tc_ptx.cuh"

#include <type_traits>

namespace sb {
namespace {

using namespace tc;

constexpr int CT = 64;                                           // tokens of a chunk
constexpr int TV = 128;                                          // value columns of a CTA
// A triangular 64 x 64 fp16 matrix [i][j], j in steps of 16: step kk holds rows 16 kk .. 63, 32 bytes each, in core matrices of 8 rows x 16
// bytes (rows 16 bytes apart, the two of a step's 16 columns 128 apart, the next 8 rows 256 apart).
constexpr int TRI_BYTES = 5120;
__host__ __device__ constexpr int tri_step(int kk) { return 32 * (64 * kk - 8 * kk * (kk - 1)); }
__device__ __forceinline__ int tri_at(int i, int j) {
    const int kk = j >> 4, r = i - 16 * kk;
    return tri_step(kk) + (r >> 3) * 256 + ((j >> 3) & 1) * 128 + (r & 7) * 16 + (j & 7) * 2;
}
// workspace of a chunk and head: T hi | T lo | M hi | (M lo) | six arrays of 64 floats | e_64, T's scale, two zeros
template <bool FINE> struct Ws {
    static constexpr int T = 0, TL = TRI_BYTES, M = 2 * TRI_BYTES, ML = 3 * TRI_BYTES, SC = (FINE ? 4 : 3) * TRI_BYTES;
    static constexpr int ER = SC, EQ = SC + 256, DK = SC + 512, OM = SC + 768, KS = SC + 1024, QS = SC + 1280, E64 = SC + 1536, TAU = SC + 1540;
    static constexpr int BYTES = SC + 1552;
};

__device__ int g_prefill_status = 0;                             // 1 + role whose wait gave up

// 128-byte rows, 16-byte pieces swizzled by the row: what SWIZZLE_128B reads
__device__ __forceinline__ uint32_t sw128(int row, int piece) { return uint32_t(row * 128 + ((piece ^ (row & 7)) << 4)); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Chunks of sequence n stand at [start / 64 + n, .. + ceil(length / 64)) of the workspace: never over those of n + 1, for any lengths.
__device__ __forceinline__ int first_chunk(const SeqRows& r, int n) { return r.start / CT + n; }

// ---------------------------------------------------------------------------------------------------- what needs no state
template <int DK, bool FINE> struct PrepSmem {
    static constexpr int TILES = 2 * CT * DK * 2, IMAGES = Ws<FINE>::BYTES, LP = CT + 4;
    __align__(1024) uint8_t a[TILES > IMAGES ? TILES : IMAGES];  // K and Q as they are, then what leaves
    __align__(16) float l[CT * LP];
    double cum[CT], low[CT];                                     // cumulative decay, and its least value so far
    float beta[CT], rk[CT], rq[CT], kk[CT], qq[CT], top[4];
};

template <typename T, int DK>
__global__ void __launch_bounds__(128) gdn_prefill_tc_prep_kernel(const shvk_gdn_seq_args a, uint8_t* __restrict__ ws) {
    constexpr bool FINE = std::is_same<T, __half>::value;
    using W = Ws<FINE>;
    using Sm = PrepSmem<DK, FINE>;
    constexpr int LP = Sm::LP;
    extern __shared__ uint8_t prep_raw[];
    Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(prep_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
    {
        const T* Q = static_cast<const T*>(a.q) + t0 * a.ldq + khead * DK;
        const T* K = static_cast<const T*>(a.k) + t0 * a.ldk + khead * DK;
        const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < CT * DK / 8 / 128; ++i) {
            const int v = tid + 128 * i, row = v / (DK / 8), p = v % (DK / 8);
            const uint32_t off = (p >> 3) * (CT * 128) + sw128(row, p & 7);
            *reinterpret_cast<uint4*>(kt + off) = row < left ? *reinterpret_cast<const uint4*>(K + row * a.ldk + p * 8) : z;
            *reinterpret_cast<uint4*>(qt + off) = row < left ? *reinterpret_cast<const uint4*>(Q + row * a.ldq + p * 8) : z;
        }
    }
    if (warp == 0) {                                             // cumulative decays in double: their differences are exponents
        double v[2], m[2];
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
        m[0] = v[0];
        m[1] = fmin(v[0], v[1]);
        double mm = m[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, mm, o);
            if (lane >= o) mm = fmin(mm, up);
        }
        const double before = __shfl_up_sync(0xffffffffu, mm, 1);
        sm.cum[2 * lane] = v[0];
        sm.cum[2 * lane + 1] = v[1];
        sm.low[2 * lane] = lane ? fmin(before, m[0]) : m[0];
        sm.low[2 * lane + 1] = lane ? fmin(before, m[1]) : m[1];
    } else if (tid >= 64) {
        const int tok = tid - 64;
        sm.beta[tok] = tok < left ? a.beta[(t0 + tok) * a.ldgb + head] : 0.0f;
    }
    __syncthreads();
    // ---------------------------------------------------------------- Gram products of the blocks (bi, bj), bj <= bi; the first is (warp, warp)
    const int g = lane >> 2, t = lane & 3, lm = lane >> 3, lr = lane & 7;
    const int blocks = warp < 2 ? 3 : 2;
    auto bi_of = [&](int b) { return b == 0 ? warp : b == 1 ? (warp == 0 ? 3 : warp == 1 ? 1 : 2) : 3; };
    auto bj_of = [&](int b) { return b == 0 ? warp : b == 1 ? (warp == 3 ? 1 : 0) : warp == 0 ? 1 : 2; };     // w0 00 30 31, w1 11 10 32, w2 22 20, w3 33 21
    float kk[3][2][4] = {}, qk[3][2][4] = {};
    const uint32_t k_s = smem_u32(kt), q_s = smem_u32(qt);
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
                ldsm4(k_s + half + sw128(rj, piece), kj);
#pragma unroll
                for (int ni = 0; ni < 2; ++ni) {
                    mma16<T>(kk[b][ni], ki, kj[ni], kj[ni + 2]);
                    mma16<T>(qk[b][ni], qi, kj[ni], kj[ni + 2]);
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
    if (tid < CT) {
        const float k2 = sm.kk[tid], rk = a.l2norm ? 1.0f / sqrtf(k2 + 1e-6f) : 1.0f;
        sm.rk[tid] = rk;
        const float len = warp_max(rk * sqrtf(k2));
        if (lane == 0) sm.top[warp] = len;
    }
    __syncthreads();
    if (tid < CT) {
        const float k2 = sm.kk[tid], q2 = sm.qq[tid], rk = sm.rk[tid];
        const float rq = a.scale * (a.l2norm ? 1.0f / sqrtf(q2 + 1e-6f) : 1.0f);
        const double cs = sm.cum[tid], last = sm.cum[CT - 1];
        const int ke = clampi(exponent_of(sqrtf(k2)), 27, 227), qe = clampi(exponent_of(sqrtf(q2)), 27, 227);
        const float e = expf(float(cs)), d = expf(float(last - cs)), kap = rk * pow2_biased(ke + 1);     // rk / ks
        sm.rq[tid] = rq;
        outf(W::KS)[tid] = pow2_biased(253 - ke);                // |ks k| < 1
        outf(W::QS)[tid] = pow2_biased(253 - qe);
        outf(W::ER)[tid] = e * kap;
        outf(W::EQ)[tid] = e * (rq * pow2_biased(qe + 1));
        outf(W::DK)[tid] = d * kap;
        // a row of M is at most |q| |k| times its largest decay
        const float most = fabsf(rq) * sqrtf(q2) * fmaxf(sm.top[0], sm.top[1]) * expf(float(cs - sm.low[tid]));
        outf(W::OM)[tid] = pow2_biased(clampi(exponent_of(most), 27, 227) + 1);
        if (tid == 0) *reinterpret_cast<float4*>(out + W::E64) = make_float4(expf(float(last)), 0.0f, 0.0f, 0.0f);
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 3; ++b) {
        if (b >= blocks) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 16 * bi_of(b) + g + 8 * h;
            const double ci = sm.cum[i];
            const float bk = sm.beta[i] * sm.rk[i], rq = sm.rq[i] * pow2_biased(254 - exponent_of(outf(W::OM)[i]));
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) {
                float m[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int j = 16 * bj_of(b) + 8 * ni + 2 * t + e;
                    const float dcy = j <= i ? expf(float(ci - sm.cum[j])) * sm.rk[j] : 0.0f;
                    sm.l[i * LP + j] = j < i ? bk * dcy * kk[b][ni][2 * h + e] : 0.0f;
                    m[e] = j <= i ? rq * dcy * qk[b][ni][2 * h + e] : 0.0f;
                }
                uint32_t mh, ml;
                split_pair(m[0], m[1], mh, ml);
                const int at = tri_at(i, 16 * bj_of(b) + 8 * ni + 2 * t);
                if (FINE) {
                    *reinterpret_cast<uint32_t*>(out + W::M + at) = mh;
                    *reinterpret_cast<uint32_t*>(out + W::ML + at) = ml;
                } else {
                    *reinterpret_cast<uint32_t*>(out + W::M + at) = pack_half(m[0], m[1]);
                }
            }
        }
    }
    __syncthreads();
    // ---------------------------------------------------------------- block column `warp` of (I + L)^-1: column 16 warp + c in lanes c, c + 16
    {
        const int c = lane & 15, half = lane >> 4;
        float x[CT], top = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d) {                            // rows 16 (warp + d) ..
            if (warp + d < 4) {
                const float* lrow = sm.l + 16 * (warp + d) * LP + 16 * warp;
                float rhs[16];
                if (d == 0) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) rhs[r] = r == c ? 1.0f : 0.0f;
                } else {
                    float acc[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {                // this half's eight rows of -sum L x
                        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                        for (int m = 0; m < 16 * d; m += 4) {
                            const float4 l = *reinterpret_cast<const float4*>(lrow + (8 * half + r) * LP + m);
                            s0 = fmaf(-l.x, x[m], s0);
                            s1 = fmaf(-l.y, x[m + 1], s1);
                            s0 = fmaf(-l.z, x[m + 2], s0);
                            s1 = fmaf(-l.w, x[m + 3], s1);
                        }
                        acc[r] = s0 + s1;
                    }
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const float other = __shfl_xor_sync(0xffffffffu, acc[r], 16);
                        rhs[r] = half ? other : acc[r];
                        rhs[8 + r] = half ? acc[r] : other;
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float s0 = rhs[i], s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
#pragma unroll
                    for (int j = 0; j < i; j += 4) {
                        const float4 l = *reinterpret_cast<const float4*>(lrow + i * LP + 16 * d + j);
                        s0 = fmaf(-l.x, x[16 * d + j], s0);
                        if (j + 1 < i) s1 = fmaf(-l.y, x[16 * d + j + 1], s1);
                        if (j + 2 < i) s2 = fmaf(-l.z, x[16 * d + j + 2], s2);
                        if (j + 3 < i) s3 = fmaf(-l.w, x[16 * d + j + 3], s3);
                    }
                    x[16 * d + i] = (s0 + s1) + (s2 + s3);
                }
            }
        }
        const float bc = sm.beta[16 * warp + c];
#pragma unroll
        for (int i = 0; i < CT; ++i)
            if (i < 16 * (4 - warp)) {
                x[i] = i < c ? 0.0f : x[i] * bc;                 // (a beta that is no number stays behind its token)
                top = fmaxf(top, fabsf(x[i]));
            }
        top = warp_max(top);
        if (lane == 0) sm.top[warp] = top;
        __syncthreads();
        top = fmaxf(fmaxf(sm.top[0], sm.top[1]), fmaxf(sm.top[2], sm.top[3]));
        const int te = clampi(exponent_of(top), 27, 227);
        const float sc = pow2_biased(253 - te);
        if (tid == 0) *outf(W::TAU) = pow2_biased(te + 1);
        uint8_t* at = out + tri_step(warp) + (c >> 3) * 128 + (c & 7) * 2;
#pragma unroll
        for (int i = 0; i < CT; ++i)
            if (i < 16 * (4 - warp) && (i & 1) == half) {
                const float v = x[i] * sc, vh = __int_as_float(__float_as_int(v) & 0xffffe000);
                *reinterpret_cast<__half*>(at + W::T + (i >> 3) * 256 + (i & 7) * 16) = __float2half_rn(vh);
                *reinterpret_cast<__half*>(at + W::TL + (i >> 3) * 256 + (i & 7) * 16) = __float2half_rn(v - vh);
            }
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(ws + ((long long)chunk * a.HV + head) * W::BYTES);
    const uint4* src = reinterpret_cast<const uint4*>(out);
    for (int i = tid; i < W::BYTES / 16; i += 128) dst[i] = src[i];
}

// ---------------------------------------------------------------------------------------------------- the walk
constexpr int COMPUTE = 8, LOADERS = 3, TC_THREADS = 32 * (COMPUTE + 1 + LOADERS);
constexpr uint32_t PREFILL_POLLS = 1u << 22;

template <int DK, bool FINE, int STAGES> struct WalkSmem {
    struct Stage {
        __align__(1024) uint8_t k[CT * DK * 2], q[CT * DK * 2];  // scaled fp16, halves of 64 keys, 128-byte rows, swizzled
        __align__(1024) uint8_t v[CT * TV * 2];                  // [token][value] as it is
        __align__(1024) uint8_t w[(Ws<FINE>::BYTES + 1023) / 1024 * 1024];
    } st[STAGES];
    __align__(16) float4 meet1[2][TV], meet2[2][TV];             // what the two threads of a value column tell each other
    __align__(8) uint64_t bars[4 * STAGES + 8];
    uint32_t tmem;
    int abort;
};

// columns of tensor memory
template <int DK> struct Cols {
    static constexpr int P = 0, S = DK, R = 2 * DK, QS = 2 * DK + 64, MU = 2 * DK + 128;     // W lies over P, D over S, U and its pieces over R
};

// D[128 x N] (+)= A (tensor memory, fp16) x B (shared memory)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)) : "memory");
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
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void pair_sync(int quad) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory"); }

template <typename T, int DK, int STAGES>
__global__ void __launch_bounds__(TC_THREADS, 1) gdn_prefill_tc_walk_kernel(const shvk_gdn_seq_args a, const uint8_t* __restrict__ ws, uint32_t polls) {
    constexpr bool FINE = std::is_same<T, __half>::value;
    using W = Ws<FINE>;
    using Sm = WalkSmem<DK, FINE, STAGES>;
    using C = Cols<DK>;
    constexpr int HALF = CT * 128;                               // bytes of 64 keys of a K or Q tile
    extern __shared__ uint8_t walk_raw[];
    Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(walk_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int splits = a.DV / TV, split = int(blockIdx.x % unsigned(splits));
    const int nh = int(blockIdx.x / unsigned(splits)), n = nh / a.HV, head = nh % a.HV, khead = head / (a.HV / a.HK);
    const SeqRows rows(a.seq_start, n, int(a.n_tokens));
    const int len = rows.end - rows.start, NB = (len + CT - 1) / CT;
    const long long in = slot_of(a.slot_in, n, a.n_slots), out = slot_of(a.slot_out, n, a.n_slots);
    const long long state_at = (long long)head * DK * a.DV + split * TV, state_of = (long long)a.HV * DK * a.DV;
    if (NB == 0) {                                               // nothing to walk: the state as it is
        if (out >= 0 && out != in)
            for (int i = tid; i < DK * TV; i += TC_THREADS) {
                const long long at = state_at + (i / TV) * (long long)a.DV + i % TV;
                a.states[out * state_of + at] = in < 0 ? 0.0f : a.states[in * state_of + at];
            }
        return;
    }
    const uint32_t bars = smem_u32(sm.bars);
    auto full = [&](int s) { return bars + 8u * s; };                                    // K, Q, V of a stage
    auto wfull = [&](int s) { return bars + 8u * (STAGES + s); };                        // T, M and scalars
    auto empty = [&](int s) { return bars + 8u * (2 * STAGES + s); };
    const uint32_t b_s = bars + 8u * (3 * STAGES), b_r = b_s + 8, b_w = b_s + 16, b_u = b_s + 24, b_d = b_s + 32, b_p = b_s + 40, b_o = b_s + 48, b_q = b_s + 56;
    if (tid == 0) {
        sm.abort = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 32 * LOADERS);
            mbar_init(wfull(s), 1);
            mbar_init(empty(s), COMPUTE + 1);
        }
        mbar_init(b_s, COMPUTE); mbar_init(b_w, COMPUTE); mbar_init(b_d, COMPUTE); mbar_init(b_q, COMPUTE);
        mbar_init(b_r, 1); mbar_init(b_u, 1); mbar_init(b_p, 1); mbar_init(b_o, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == COMPUTE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abortp = &sm.abort;
    // A role whose wait has given up goes on through its loop without waiting, issuing or writing, so that the barriers among warps are
    // met by all; the others' waits end with the flag.
    bool dead = false;
    auto wait = [&](uint32_t bar, uint32_t parity) {
        const bool gave_up = !dead && !mbar_wait(bar, parity & 1u, abortp, polls);
        if (__any_sync(0xffffffffu, gave_up)) {
            dead = true;
            *abortp = 1;
            atomicCAS(&g_prefill_status, 0, 1 + (warp < COMPUTE ? 0 : warp == COMPUTE ? 1 : 2));
        }
    };

    if (warp < COMPUTE) {
        // ------------------------------------------------------------------------------------------- the value columns
        constexpr int KH = DK / 2;                               // keys of a thread
        const int quad = warp & 3, half = warp >> 2, row = 32 * quad + lane;
        const uint32_t tl = tmem + (uint32_t(32 * quad) << 16);
        float S[KH], sig = 1.0f, inv = 1.0f, mine = 0.0f;       // S in units of inv; mine: the largest |S| here
        {
            const float* src = a.states + (in < 0 ? 0 : in) * state_of + state_at + (long long)(half * KH) * a.DV + row;
#pragma unroll
            for (int i = 0; i < KH; ++i) {
                S[i] = in < 0 ? 0.0f : src[i * (long long)a.DV];
                mine = fmaxf(mine, fabsf(S[i]));
            }
            sm.meet1[half][row] = make_float4(mine, 0.0f, 0.0f, 0.0f);
            pair_sync(quad);
            const float m = fmaxf(mine, sm.meet1[half ^ 1][row].x);
            const int b = m > 0.0f ? clampi(265 - exponent_of(m), 27, 191) : 127;        // m sig in [2^11, 2^12)
            sig = pow2_biased(b);
            inv = pow2_biased(254 - b);
#pragma unroll
            for (int i = 0; i < KH; ++i) S[i] *= sig;
            mine *= sig;
            pair_sync(quad);                                     // meet1 is read
        }
        auto give_state = [&]() {                                // pieces of S to tensor memory
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
        };
        give_state();
        for (int c = 0; c < NB; ++c) {
            const int s = c % STAGES;
            const typename Sm::Stage& st = sm.st[s];
            const uint32_t ph = uint32_t(c) & 1u, sph = uint32_t(c / STAGES) & 1u;
            const float* sc = reinterpret_cast<const float*>(st.w);
            auto four = [&](int at, int i) { return *reinterpret_cast<const float4*>(sc + at / 4 + 32 * half + i); };
            wait(wfull(s), sph);
            wait(full(s), sph);
            wait(b_r, ph);
            tc_fence_after();
            // ------------------------------------------------------------------- W = V - e K S0 of this half's 32 tokens
            float x[32], most = 0.0f, sound = 0.0f;
            {
                const T* v = reinterpret_cast<const T*>(st.v) + 32 * half * TV + row;
                uint32_t r[32];
                tc_ld32(tl + C::R + 32 * half, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 er = four(W::ER, i);
                    const float e[4] = {er.x, er.y, er.z, er.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        x[i + u] = fmaf(-e[u], __uint_as_float(r[i + u]), to_float(v[(i + u) * TV]) * sig);
                        most = fmaxf(most, fabsf(x[i + u]));
                        sound += x[i + u];
                    }
                }
            }
            // What is no number, or none any more, belongs to its own token and those behind it, but a product's zeros in front of it
            // spread it over the whole chunk: a column goes on with zeros from its first bad token on, and is marked from there on.
            int first = CT;
            auto find_bad = [&](const float (&y)[32]) {
#pragma unroll
                for (int i = 31; i >= 0; --i)
                    if (!(fabsf(y[i]) <= 3.402823466e38f)) first = min(first, 32 * half + i);
            };
            auto cut = [&](float (&y)[32]) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (32 * half + i >= first) y[i] = 0.0f;
            };
            if (!(fabsf(sound) <= 3.402823466e38f)) {
                find_bad(x);
                most = 0.0f;                                     // of the others: an infinity sets no scale
#pragma unroll
                for (int i = 0; i < 32; ++i) most = fmaxf(most, fabsf(x[i]) <= 3.402823466e38f ? fabsf(x[i]) : 0.0f);
            }
            sm.meet1[half][row] = make_float4(most, mine, __int_as_float(first), 0.0f);
            pair_sync(quad);
            const float4 other = sm.meet1[half ^ 1][row];
            first = min(first, __float_as_int(other.z));
            if (first < CT) cut(x);
            const float stop = fmaxf(mine, other.y);             // the column's largest |S|
            const int wb = clampi(exponent_of(fmaxf(most, other.x)), 27, 227);
            const float wsc = pow2_biased(261 - wb);             // W within 2^8, so that U, a sum of 64, is within 2^14
            {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) split_pair(x[2 * i] * wsc, x[2 * i + 1] * wsc, hi[i], lo[i]);
                tc_st16(tl + C::P + 16 * half, hi);
                tc_st16(tl + C::P + 32 + 16 * half, lo);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_w);
            const float uf = pow2_biased(wb - 7) * *reinterpret_cast<const float*>(st.w + W::TAU);
            wait(b_u, ph);
            tc_fence_after();
            // ------------------------------------------------------------------- D = exp(c_64 - c_j) U, in the state's units
            float sum = 0.0f, f = 1.0f;
            const float e64 = *reinterpret_cast<const float*>(st.w + W::E64);
            {
                uint32_t r[32];
                tc_ld32(tl + C::R + 32 * half, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 dk = four(W::DK, i);
                sum += (fabsf(x[i] * (uf * dk.x)) + fabsf(x[i + 1] * (uf * dk.y))) + (fabsf(x[i + 2] * (uf * dk.z)) + fabsf(x[i + 3] * (uf * dk.w)));
            }
            if (!(sum <= 3.402823466e38f)) find_bad(x);
            sm.meet2[half][row] = make_float4(sum, __int_as_float(first), 0.0f, 0.0f);
            pair_sync(quad);
            {
                const float4 o2 = sm.meet2[half ^ 1][row];
                first = min(first, __float_as_int(o2.y));
                const float top = fmaf(e64, stop, sum + o2.x);   // bounds the new |S|: |k| < 1 in its units
                if (!(top <= 32768.0f && (top >= 512.0f || top == 0.0f))) {
                    const int b = exponent_of(sig);
                    const int nb = top > 0.0f ? clampi(b + clampi(138 - exponent_of(top), -100, 100), 27, 191) : b;     // top f in [2^11, 2^12)
                    f = pow2_biased(127 + clampi(nb - b, -120, 120));
                }
            }
            if (first < CT) cut(x);
            {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (FINE) split_pair(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
                    else hi[i] = pack_half(x[2 * i], x[2 * i + 1]);
                }
                tc_st16(tl + C::R + 32 * half, hi);              // over the U that this warp has read
                if (FINE) tc_st16(tl + C::R + 32 * half + 16, lo);
                const float nan = __int_as_float(0x7fffffff), fu = first < CT ? nan : f * uf;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 dk = four(W::DK, i);
                    split_pair(x[i] * (fu * dk.x), x[i + 1] * (fu * dk.y), hi[i / 2], lo[i / 2]);
                    split_pair(x[i + 2] * (fu * dk.z), x[i + 3] * (fu * dk.w), hi[i / 2 + 1], lo[i / 2 + 1]);
                }
                tc_st16(tl + C::S + 16 * half, hi);
                tc_st16(tl + C::S + 32 + 16 * half, lo);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_d);
            wait(b_p, ph);
            tc_fence_after();
            // ------------------------------------------------------------------- S = e_64 S0 + K^T D
            const float ef = e64 * f, was = inv;
            mine = 0.0f;
#pragma unroll
            for (int p = 0; p < KH / 32; ++p) {
                uint32_t r[32];
                tc_ld32(tl + C::P + half * KH + 32 * p, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 v = fma2(make_float2(ef, ef), make_float2(S[32 * p + i], S[32 * p + i + 1]), make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
                    S[32 * p + i] = v.x;
                    S[32 * p + i + 1] = v.y;
                    mine = fmaxf(mine, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            }
            sig *= f;
            inv = pow2_biased(254 - exponent_of(sig));
            if (c + 1 < NB) give_state();
            // ------------------------------------------------------------------- O = M U + e Q S0
            wait(b_o, ph);
            tc_fence_after();
            {
                uint32_t q[32], m[32];
                tc_ld32(tl + C::QS + 32 * half, q);
                tc_ld32(tl + C::MU + 32 * half, m);
                tc_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b_q);
                T* o = static_cast<T*>(a.o) + (rows.start + c * CT + 32 * half) * a.ldo + (long long)head * a.DV + split * TV + row;
                const int left = dead ? 0 : len - c * CT - 32 * half;
                const float fo = was * uf;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 om = four(W::OM, i), eq = four(W::EQ, i);
                    const float omv[4] = {om.x, om.y, om.z, om.w}, eqv[4] = {eq.x, eq.y, eq.z, eq.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        float y = fmaf(__uint_as_float(m[i + u]) * fo, omv[u], was * (eqv[u] * __uint_as_float(q[i + u])));
                        if (32 * half + i + u >= first) y = __int_as_float(0x7fffffff);
                        if (i + u < left) o[(i + u) * a.ldo] = from_float<T>(y);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(s));
        }
        if (out >= 0 && !dead) {
            float* dst = a.states + out * state_of + state_at + (long long)(half * KH) * a.DV + row;
#pragma unroll
            for (int i = 0; i < KH; ++i) dst[i * (long long)a.DV] = S[i] * inv;
        }
    } else if (warp == COMPUTE) {
        // ------------------------------------------------------------------------------------------- the products
        for (int c = 0; c < NB; ++c) {
            const int s = c % STAGES;
            const uint32_t ph = uint32_t(c) & 1u, sph = uint32_t(c / STAGES) & 1u;
            const uint32_t kt = smem_u32(sm.st[s].k), qt = smem_u32(sm.st[s].q), wt = smem_u32(sm.st[s].w);
            constexpr uint32_t id64 = idesc_f16(64, false);
            wait(full(s), sph);
            wait(b_s, ph);
            if (c > 0) wait(b_o, ph ^ 1u);                       // M U has read the pieces of U that K S0 overwrites
            tc_fence_after();
            if (!dead && elect_one()) {
#pragma unroll
                for (int p = 0; p < DK / 16; ++p) {
                    const uint64_t b = smem_desc_sw128(kt + (p >> 2) * HALF) + uint64_t(2 * (p & 3));
                    mma_ts(tmem + C::R, tmem + C::S + 8 * p, b, id64, p > 0);
                    mma_ts(tmem + C::R, tmem + C::S + DK / 2 + 8 * p, b, id64, true);
                }
                tc_commit(b_r);
            }
            __syncwarp();
            if (c > 0) wait(b_q, ph ^ 1u);                       // the last chunk's outputs are read
            tc_fence_after();
            if (!dead && elect_one()) {
#pragma unroll
                for (int p = 0; p < DK / 16; ++p) {
                    const uint64_t b = smem_desc_sw128(qt + (p >> 2) * HALF) + uint64_t(2 * (p & 3));
                    mma_ts(tmem + C::QS, tmem + C::S + 8 * p, b, id64, p > 0);
                    if (FINE) mma_ts(tmem + C::QS, tmem + C::S + DK / 2 + 8 * p, b, id64, true);
                }
            }
            __syncwarp();
            wait(wfull(s), sph);
            wait(b_w, ph);
            tc_fence_after();
            if (!dead && elect_one()) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {                 // T is triangular: tokens 16 kk .. reach columns 16 kk .. 63
                    const uint64_t th = desc_plain(wt + W::T + tri_step(kk), 128, 256), tlo = desc_plain(wt + W::TL + tri_step(kk), 128, 256);
                    const uint32_t id = idesc_f16(64 - 16 * kk, false), d = tmem + C::R + 16 * kk;
                    mma_ts(d, tmem + C::P + 8 * kk, th, id, kk > 0);
                    mma_ts(d, tmem + C::P + 8 * kk, tlo, id, true);
                    mma_ts(d, tmem + C::P + 32 + 8 * kk, th, id, true);
                }
                tc_commit(b_u);
            }
            __syncwarp();
            wait(b_d, ph);
            tc_fence_after();
            if (!dead && elect_one()) {
                constexpr uint32_t idk = idesc_f16(DK, true);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint64_t b = desc_mn(kt + 2048 * kk, HALF);
                    mma_ts(tmem + C::P, tmem + C::S + 8 * kk, b, idk, kk > 0);
                    mma_ts(tmem + C::P, tmem + C::S + 32 + 8 * kk, b, idk, true);
                }
                tc_commit(b_p);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint64_t mh = desc_plain(wt + W::M + tri_step(kk), 128, 256);
                    const uint32_t id = idesc_f16(64 - 16 * kk, false), d = tmem + C::MU + 16 * kk, u = tmem + C::R + 32 * (kk >> 1) + 8 * (kk & 1);
                    mma_ts(d, u, mh, id, kk > 0);
                    if (FINE) {
                        mma_ts(d, u, desc_plain(wt + W::ML + tri_step(kk), 128, 256), id, true);
                        mma_ts(d, u + 16, mh, id, true);
                    }
                }
                tc_commit(b_o);
                tc_commit(empty(s));
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------------------------------------- the operands
        const int lt = tid - 32 * (COMPUTE + 1);
        constexpr int NT = 32 * LOADERS, KALL = CT * DK / 8, KN = (KALL + NT - 1) / NT, VALL = CT * TV / 8;
        const T* Q = static_cast<const T*>(a.q) + rows.start * a.ldq + khead * DK;
        const T* K = static_cast<const T*>(a.k) + rows.start * a.ldk + khead * DK;
        const T* V = static_cast<const T*>(a.v) + rows.start * a.ldv + (long long)head * a.DV + split * TV;
        const uint8_t* src = ws + ((long long)first_chunk(rows, n) * a.HV + head) * W::BYTES;
        const uint4 z = make_uint4(0, 0, 0, 0);
        for (int c = 0; c < NB; ++c) {
            const int s = c % STAGES;
            typename Sm::Stage& st = sm.st[s];
            const uint32_t sph = uint32_t(c / STAGES) & 1u;
            const int left = len - c * CT;
            uint4 k[KN], q[KN];
#pragma unroll
            for (int i = 0; i < KN; ++i) {
                const int x = lt + NT * i, row = x / (DK / 8), p = x % (DK / 8);
                const bool has = x < KALL && row < left;
                k[i] = has ? *reinterpret_cast<const uint4*>(K + (c * CT + row) * a.ldk + p * 8) : z;
                q[i] = has ? *reinterpret_cast<const uint4*>(Q + (c * CT + row) * a.ldq + p * 8) : z;
            }
            wait(empty(s), sph ^ 1u);
            if (lt == 0 && !dead) {
                mbar_expect_tx(wfull(s), W::BYTES);
                bulk_load(smem_u32(st.w), src + (long long)c * a.HV * W::BYTES, W::BYTES, wfull(s));
            }
            for (int x = lt; x < VALL; x += NT) {
                const int row = x / (TV / 8), p = x % (TV / 8), has = row < left ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(st.v) + row * (TV * 2) + p * 16),
                             "l"(has ? static_cast<const void*>(V + (c * CT + row) * a.ldv + p * 8) : src), "r"(has) : "memory");
            }
            wait(wfull(s), sph);
            const float* ks = reinterpret_cast<const float*>(st.w + W::KS);
            const float* qs = reinterpret_cast<const float*>(st.w + W::QS);
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
#pragma unroll
            for (int i = 0; i < KN; ++i) {
                const int x = lt + NT * i, row = x / (DK / 8), p = x % (DK / 8);
                if (x >= KALL) break;
                const uint32_t off = (p >> 3) * HALF + sw128(row, p & 7);
                *reinterpret_cast<uint4*>(st.k + off) = turn(k[i], ks[row]);
                *reinterpret_cast<uint4*>(st.q + off) = turn(q[i], qs[row]);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async();
            mbar_arrive(full(s));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abortp) {                                               // products may still be on their way: a millisecond is a thousand times theirs
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    tc_fence_after();
    if (warp == COMPUTE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <typename T, int DK> int launch_tc(const shvk_gdn_seq_args& a, uint8_t* ws, cudaStream_t s) {
    constexpr bool FINE = std::is_same<T, __half>::value;
    constexpr int STAGES = 2;
    const long long items = (a.n_tokens / CT + a.n_seq + 1) * a.HV, ctas = (long long)a.n_seq * a.HV * (a.DV / TV);
    if (items > 0x7fffffff || ctas > 0x7fffffff) return int(cudaErrorInvalidValue);
    if (a.n_tokens > 0) {
        constexpr int smem = int(sizeof(PrepSmem<DK, FINE>)) + 1024;
        const cudaError_t e = cudaFuncSetAttribute(gdn_prefill_tc_prep_kernel<T, DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return int(e);
        gdn_prefill_tc_prep_kernel<T, DK><<<unsigned(items), 128, smem, s>>>(a, ws);
        if (const cudaError_t le = cudaGetLastError(); le != cudaSuccess) return int(le);
    }
    constexpr int smem = int(sizeof(WalkSmem<DK, FINE, STAGES>)) + 1024;
    static_assert(smem <= 227 * 1024, "the stages fit");
    const cudaError_t e = cudaFuncSetAttribute(gdn_prefill_tc_walk_kernel<T, DK, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return int(e);
    gdn_prefill_tc_walk_kernel<T, DK, STAGES><<<unsigned(ctas), TC_THREADS, smem, s>>>(a, ws, PREFILL_POLLS);
    return int(cudaGetLastError());
}

}  // namespace

size_t gdn_prefill_tc_workspace(const shvk_gdn_seq_args& a) {
    return size_t(a.n_tokens / CT + a.n_seq + 1) * size_t(a.HV) * size_t(a.dtype == DT_F16 ? Ws<true>::BYTES : Ws<false>::BYTES);
}
int gdn_prefill_tc(const shvk_gdn_seq_args& a, uint8_t* ws, cudaStream_t s) {
    if (a.dtype == DT_BF16) return a.DK == 64 ? launch_tc<__nv_bfloat16, 64>(a, ws, s) : launch_tc<__nv_bfloat16, 128>(a, ws, s);
    return a.DK == 64 ? launch_tc<__half, 64>(a, ws, s) : launch_tc<__half, 128>(a, ws, s);
}

}  // namespace sb

extern "C" int shvk_gdn_prefill_status(int* status_out) {
    if (!status_out) return int(cudaErrorInvalidValue);
    return int(cudaMemcpyFromSymbol(status_out, sb::g_prefill_status, sizeof(int)));
}
