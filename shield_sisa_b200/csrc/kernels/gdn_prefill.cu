// The gated delta rule over packed sequences in chunks of 16 tokens, states taken from a pool's slots and left in them (see the header
// for the arguments).  Per chunk, with c_i the chunk's cumulative log decay, e_i = exp(c_i), and S0 the state that enters it:
//
//     L_ij = beta_i exp(c_i - c_j) (k_i . k_j)  (j < i),  T = (I + L)^-1 diag(beta),  M_ij = exp(c_i - c_j) (q_i . k_j)  (j <= i)
//     U = T (V - diag(e) K S0),  O = M U + diag(e) Q S0,  S = e_16 S0 + K^T diag(exp(c_16 - c_j)) U
// T and M do not depend on the state: one kernel makes them for all chunks at once (and the row scales below), a second walks each
// head's chunks with its state in registers.
//
// Precision.  The state that a call leaves is held to float32, which one rounding of an operand to 16 bits on the way would lose.  The
// tensor cores multiply 16-bit pieces: an operand on the state's way is two fp16 pieces (22 bits), and the products that matter, hi hi +
// hi lo + lo hi, are summed in float32.  K and Q are 16-bit values already: one piece.  fp16 has the bits (bf16 pieces would have to be
// three) but not the range, so everything is scaled by powers of two, which cost no bits: a token's k and q by their norms, T by its
// largest entry, rows of M by theirs, and the rows of S^T, W^T, U^T (one value column each; what a chunk does to them is linear) by scales
// that the walk keeps or finds anew.  On the output's way S, M and U are two pieces as well (with one, of eleven bits, 11 % of bf16
// outputs were not the rule's value rounded, now 0.03 %, in gdn_prefill_tc.cu 0.12 %; it costs 4 % of the time here, 6 % there).  Sums over
// tokens that last, S = e S + P, are rounded float32 FMAs and not tensor-core accumulations, whose truncation would lean one way for
// thousands of chunks.
//
// This form takes short sequences and the widths that fill no CTA of gdn_prefill_tc.cu (see takes_tc).  128 sequences of 48 tokens, 6 heads of
// 128 x 128, bf16: 80 us, for 38 MB of rows and 100 MB of states (21 us).  The walk's chain binds, dependent products and exchanges among
// lanes: a chunk of 16 tokens takes 1.2 to 1.6 us (8 sequences of 2,048 tokens, DK 64, DV 64: 205 us).
#include "gdn_pieces.cuh"
#include "gdn_seq.cuh"

#include <type_traits>

namespace sb {
namespace {

constexpr int PB = 16;                                          // tokens of a chunk
// workspace of a chunk and head: T hi | T lo | M hi | M lo (fp16 16 x 16) | six arrays of 16 floats | e_16 and T's scale
constexpr int PW_T = 0, PW_TL = 512, PW_M = 1024, PW_ML = 1536, PW_ER = 2048, PW_EQ = 2112, PW_DK = 2176, PW_OM = 2240, PW_KS = 2304, PW_QS = 2368,
              PW_E16 = 2432, PW_TAU = 2436, PW_BYTES = 2448;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {      // bytes 16, or 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void stsm4t(uint32_t addr, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}

// Rows of ROWB bytes, 16-byte pieces swizzled so that the same piece of eight successive rows lies in eight different bank groups.
template <int ROWB> __device__ __forceinline__ uint32_t tile_off(int row, int piece) {
    constexpr int PER = ROWB / 16;                              // pieces of a row
    if constexpr (PER >= 8) return uint32_t(row * ROWB + ((piece ^ (row & 7)) << 4));
    else return uint32_t(row * ROWB + ((piece ^ ((row / (8 / PER)) & (PER - 1))) << 4));
}

// Chunks of sequence n stand at [start / 16 + n, .. + ceil(length / 16)) of the workspace: never over those of n + 1, for any lengths.
__device__ __forceinline__ int first_chunk(const SeqRows& r, int n) { return r.start / PB + n; }

// ---------------------------------------------------------------------------------------------------- what needs no state
template <int DK> struct PrepWarp {
    __align__(16) uint8_t k[PB * DK * 2], q[PB * DK * 2];
    __align__(16) float lf[2][PB * (PB + 4)];
    double cum[PB];
    float beta[2][PB], rk[PB], rq[PB], kk[PB], qq[PB];
    __align__(16) uint8_t out[2][PW_BYTES];
};

// A warp makes two (chunk, head)s, the triangular inverses of both at once on its two halves.
template <typename T, int DK>
__global__ void __launch_bounds__(128, 4) gdn_prefill_prep_kernel(const shvk_gdn_seq_args a, uint8_t* __restrict__ ws, long long items) {
    constexpr int ROWB = DK * 2, VPR = DK / 8, KSTEP = DK / 16, VEC = PB * VPR / 32, LP = PB + 4;
    extern __shared__ __align__(16) uint8_t prep_raw[];
    last_is_done();
    next_may_start();                                            // (behind the wait: the walk reads where sequences lie before its own)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    PrepWarp<DK>& sm = reinterpret_cast<PrepWarp<DK>*>(prep_raw)[warp];
    const long long item0 = ((long long)blockIdx.x * 4 + warp) * 2;
    const int g = lane >> 2, t = lane & 3, lm = lane >> 3, lr = lane & 7;
    bool live[2] = {false, false};
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
        const long long item = item0 + slot;
        if (item >= items) break;
        const int chunk = int(item / a.HV), head = int(item % a.HV), khead = head / (a.HV / a.HK);
        // the last sequence whose first chunk is not behind this one
        int n = 0;
        for (int lo = 0, hi = a.n_seq - 1; lo <= hi;) {
            const int mid = (lo + hi) >> 1;
            if (first_chunk(SeqRows(a.seq_start, mid, int(a.n_tokens)), mid) <= chunk) { n = mid; lo = mid + 1; } else hi = mid - 1;
        }
        const SeqRows rows(a.seq_start, n, int(a.n_tokens));
        const int t0 = rows.start + (chunk - first_chunk(rows, n)) * PB, left = rows.end - t0;
        if (t0 < rows.start || left <= 0) continue;             // no chunk of any sequence stands here
        live[slot] = true;
        const T* Q = static_cast<const T*>(a.q) + t0 * a.ldq + khead * DK;
        const T* K = static_cast<const T*>(a.k) + t0 * a.ldk + khead * DK;
        const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int v = lane + 32 * i, row = v / VPR, c = v % VPR;
            const uint4 kv = row < left ? *reinterpret_cast<const uint4*>(K + row * a.ldk + c * 8) : z;
            const uint4 qv = row < left ? *reinterpret_cast<const uint4*>(Q + row * a.ldq + c * 8) : z;
            *reinterpret_cast<uint4*>(sm.k + tile_off<ROWB>(row, c)) = kv;
            *reinterpret_cast<uint4*>(sm.q + tile_off<ROWB>(row, c)) = qv;
        }
        const int tok = lane & (PB - 1);
        float dec = tok < left ? a.g[(t0 + tok) * a.ldgb + head] : 0.0f;
        const float bt = tok < left ? a.beta[(t0 + tok) * a.ldgb + head] : 0.0f;
        dec = dec < -1000.0f ? -1000.0f : dec;                   // exp(-1000) = 0, and no difference of two infinities (NaN stays)
        // cumulative decays in double: differences of far apart ones are exponents
        double cs = dec;
#pragma unroll
        for (int o = 1; o < PB; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, cs, o);
            if (tok >= o) cs += up;
        }
        const double last = __shfl_sync(0xffffffffu, cs, PB - 1);
        if (lane < PB) {
            sm.cum[tok] = cs;
            sm.beta[slot][tok] = bt;
        }
        __syncwarp();
        // K K^T, Q K^T and the diagonal of Q Q^T
        float kk[2][4] = {}, qk[2][4] = {}, qq[2][4] = {};
        const uint32_t k_s = smem_u32(sm.k), q_s = smem_u32(sm.q);
#pragma unroll
        for (int p = 0; p < KSTEP; ++p) {
            const uint32_t off = tile_off<ROWB>((lm & 1) * 8 + lr, 2 * p + (lm >> 1));
            uint32_t kf[4], qf[4];
            ldsm4(k_s + off, kf);
            ldsm4(q_s + off, qf);
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) {
                mma16<T>(kk[ni], kf, kf[ni], kf[ni + 2]);
                mma16<T>(qk[ni], qf, kf[ni], kf[ni + 2]);
                mma16<T>(qq[ni], qf, qf[ni], qf[ni + 2]);
            }
        }
        if ((g >> 1) == t) {                                     // [ni][2 ni + e] of lane (g, t): entry (8 ni + g, 8 ni + 2 t + e)
            const int e = g & 1;
            sm.kk[g] = e ? kk[0][1] : kk[0][0];
            sm.kk[8 + g] = e ? kk[1][3] : kk[1][2];
            sm.qq[g] = e ? qq[0][1] : qq[0][0];
            sm.qq[8 + g] = e ? qq[1][3] : qq[1][2];
        }
        __syncwarp();
        uint8_t* out = sm.out[slot];
        auto outf = [&](int at) { return reinterpret_cast<float*>(out + at); };
        if (lane < PB) {
            const float k2 = sm.kk[tok], q2 = sm.qq[tok];
            const float rk = a.l2norm ? 1.0f / sqrtf(k2 + 1e-6f) : 1.0f, rq = a.scale * (a.l2norm ? 1.0f / sqrtf(q2 + 1e-6f) : 1.0f);
            const int ke = clampi(exponent_of(sqrtf(k2)), 27, 227), qe = clampi(exponent_of(sqrtf(q2)), 27, 227);
            const float e = expf(float(cs)), d = expf(float(last - cs)), kap = rk * pow2_biased(ke + 1);     // rk / ks
            sm.rk[tok] = rk;
            sm.rq[tok] = rq;
            outf(PW_KS)[tok] = pow2_biased(253 - ke);            // |ks k| < 1
            outf(PW_QS)[tok] = pow2_biased(253 - qe);
            outf(PW_ER)[tok] = e * kap;
            outf(PW_EQ)[tok] = e * (rq * pow2_biased(qe + 1));
            outf(PW_DK)[tok] = d * kap;
            if (tok == 0) *outf(PW_E16) = expf(float(last));
        }
        __syncwarp();
        float* lf = sm.lf[slot];
        uint32_t* mh = reinterpret_cast<uint32_t*>(out + PW_M);  // eight words a row
        uint32_t* ml = reinterpret_cast<uint32_t*>(out + PW_ML);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                            // rows g and g + 8
            const int i = g + 8 * h;
            float m[2][2], top = 0.0f;
#pragma unroll
            for (int ni = 0; ni < 2; ++ni)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int j = 8 * ni + 2 * t + e;
                    const float dcy = j <= i ? expf(float(sm.cum[i] - sm.cum[j])) * sm.rk[j] : 0.0f;
                    lf[i * LP + j] = j < i ? sm.beta[slot][i] * sm.rk[i] * dcy * kk[ni][2 * h + e] : 0.0f;
                    m[ni][e] = j <= i ? sm.rq[i] * dcy * qk[ni][2 * h + e] : 0.0f;
                    top = fmaxf(top, fabsf(m[ni][e]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int me = clampi(exponent_of(top), 27, 227);
            const float sc = pow2_biased(253 - me);              // the row's entries below one
            if (t == 0) outf(PW_OM)[i] = pow2_biased(me + 1);
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) split_pair(m[ni][0] * sc, m[ni][1] * sc, mh[i * 8 + 4 * ni + t], ml[i * 8 + 4 * ni + t]);
        }
        __syncwarp();
    }
    {                                                            // column `col` of (I + L)^-1 by forward substitution, a half-warp each
        const int slot = lane >> 4, col = lane & (PB - 1);
        const bool on = slot ? live[1] : live[0];
        const float* lf = sm.lf[slot];
        float x[PB], top = 0.0f;
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            float s0 = i == col ? 1.0f : 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const float4 l = *reinterpret_cast<const float4*>(lf + i * LP + j);
                s0 = fmaf(-l.x, x[j], s0);
                if (j + 1 < i) s1 = fmaf(-l.y, x[j + 1], s1);
                if (j + 2 < i) s2 = fmaf(-l.z, x[j + 2], s2);
                if (j + 3 < i) s3 = fmaf(-l.w, x[j + 3], s3);
            }
            x[i] = (s0 + s1) + (s2 + s3);
        }
        const float bc = sm.beta[slot][col];
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            x[i] = i < col ? 0.0f : x[i] * bc;                   // (a beta that is no number stays behind its token)
            top = fmaxf(top, fabsf(x[i]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int te = clampi(exponent_of(top), 27, 227);
        const float sc = pow2_biased(253 - te);
        if (on) {
            __half* th = reinterpret_cast<__half*>(sm.out[slot] + PW_T);
            __half* tl = reinterpret_cast<__half*>(sm.out[slot] + PW_TL);
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const float v = x[i] * sc, vh = __int_as_float(__float_as_int(v) & 0xffffe000);
                th[i * PB + col] = __float2half_rn(vh);
                tl[i * PB + col] = __float2half_rn(v - vh);
            }
            if (col == 0) {
                *reinterpret_cast<float*>(sm.out[slot] + PW_TAU) = pow2_biased(te + 1);
                *reinterpret_cast<float2*>(sm.out[slot] + PW_TAU + 4) = make_float2(0.0f, 0.0f);
            }
        }
    }
    __syncwarp();
#pragma unroll
    for (int slot = 0; slot < 2; ++slot) {
        if (!live[slot]) continue;
        uint4* dst = reinterpret_cast<uint4*>(ws + (item0 + slot) * PW_BYTES);
        const uint4* src = reinterpret_cast<const uint4*>(sm.out[slot]);
        for (int i = lane; i < PW_BYTES / 16; i += 32) dst[i] = src[i];
    }
}

// ---------------------------------------------------------------------------------------------------- the walk
// A chunk's operands in shared memory.  K and Q arrive in the caller's type and are turned in place into scaled fp16.
template <int DK, int VC> struct Stage {
    __align__(128) uint8_t k[PB * DK * 2], q[PB * DK * 2], v[PB * VC * 2];
    __align__(16) uint8_t w[PW_BYTES];
};
template <int DK, int VC, int NSLOT> struct ScanSmem {
    Stage<DK, VC> st[NSLOT];
    __align__(128) uint8_t o[2][PB * VC * 2];                    // finished rows in the caller's type
};

// NW warps, 16 value columns each: a CTA has VC = 16 NW of the head's DV.  The values are the rows of the products (S^T, U^T: M = 16),
// so that what one product leaves in registers is the next one's operand as it lies.
template <typename T, int DK, int NW, int NSLOT>
__global__ void __launch_bounds__(NW * 32, 1) gdn_prefill_scan_kernel(const shvk_gdn_seq_args a, const uint8_t* __restrict__ ws) {
    constexpr int VC = 16 * NW, NT = NW * 32, KSTEP = DK / 16, NJ = DK / 8, ROWB = DK * 2, VROWB = VC * 2, VPR = DK / 8, VPV = VC / 8;
    constexpr int KN = PB * VPR, VN = PB * VPV, WN = PW_BYTES / 16;
    extern __shared__ __align__(128) uint8_t scan_raw[];
    ScanSmem<DK, VC, NSLOT>& sm = *reinterpret_cast<ScanSmem<DK, VC, NSLOT>*>(scan_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3, lm = lane >> 3, lr = lane & 7;
    const int splits = a.DV / VC, split = blockIdx.x % splits;
    const int nh = blockIdx.x / splits, n = nh / a.HV, head = nh % a.HV, khead = head / (a.HV / a.HK);
    const SeqRows rows(a.seq_start, n, int(a.n_tokens));
    const int len = rows.end - rows.start, NB = (len + PB - 1) / PB;
    const long long in = slot_of(a.slot_in, n, a.n_slots), out = slot_of(a.slot_out, n, a.n_slots);
    if (len == 0 && (out < 0 || out == in)) {
        last_is_done();
        return;
    }
    const int col0 = split * VC + warp * 16;                     // the warp's first value column
    const T* Q = static_cast<const T*>(a.q) + rows.start * a.ldq + khead * DK;
    const T* K = static_cast<const T*>(a.k) + rows.start * a.ldk + khead * DK;
    const T* V = static_cast<const T*>(a.v) + rows.start * a.ldv + (long long)head * a.DV + split * VC;
    T* O = static_cast<T*>(a.o) + rows.start * a.ldo + (long long)head * a.DV + split * VC;
    const uint8_t* W = ws + ((long long)first_chunk(rows, n) * a.HV + head) * PW_BYTES;

    auto issue = [&](int c) {                                    // copies of chunk c; rows past the sequence are zeros
        if (c < NB) {
            Stage<DK, VC>& st = sm.st[c % NSLOT];
            const int left = len - c * PB;
            const uint8_t* w = W + (long long)c * a.HV * PW_BYTES;
#pragma unroll
            for (int i = tid; i < KN; i += NT) {
                const int row = i / VPR, p = i % VPR, has = row < left ? 16 : 0;
                const uint32_t off = tile_off<ROWB>(row, p);
                cp_async16(smem_u32(st.k) + off, has ? static_cast<const void*>(K + (c * PB + row) * a.ldk + p * 8) : w, has);
                cp_async16(smem_u32(st.q) + off, has ? static_cast<const void*>(Q + (c * PB + row) * a.ldq + p * 8) : w, has);
            }
#pragma unroll
            for (int i = tid; i < VN; i += NT) {
                const int row = i / VPV, p = i % VPV, has = row < left ? 16 : 0;
                cp_async16(smem_u32(st.v) + tile_off<VROWB>(row, p), has ? static_cast<const void*>(V + (c * PB + row) * a.ldv + p * 8) : w, has);
            }
            for (int i = tid; i < WN; i += NT) cp_async16(smem_u32(st.w) + i * 16, w + i * 16, 16);
        }
        cp_commit();                                             // an empty group past the end keeps the count in step
    };
    auto convert = [&](int c) {                                  // chunk c's K and Q, landed, to scaled fp16
        if (c >= NB) return;
        Stage<DK, VC>& st = sm.st[c % NSLOT];
#pragma unroll
        for (int i = tid; i < 2 * KN; i += NT) {
            const int j = i % KN, row = j / VPR, p = j % VPR;
            uint4* at = reinterpret_cast<uint4*>((i < KN ? st.k : st.q) + tile_off<ROWB>(row, p));
            const float sc = reinterpret_cast<const float*>(st.w + (i < KN ? PW_KS : PW_QS))[row];
            uint4 x = *at;
            uint32_t* e = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const T* two = reinterpret_cast<const T*>(&e[u]);
                const float2 v = mul2(make_float2(to_float(two[0]), to_float(two[1])), make_float2(sc, sc));
                e[u] = pack_half(v.x, v.y);
            }
            *at = x;
        }
    };
    auto store_rows = [&](int c) {                               // finished rows of chunk c
        const uint8_t* o = sm.o[c & 1];
        const int left = len - c * PB;
#pragma unroll
        for (int i = tid; i < VN; i += NT) {
            const int row = i / VPV, p = i % VPV;
            if (row < left) *reinterpret_cast<uint4*>(O + (c * PB + row) * a.ldo + p * 8) = *reinterpret_cast<const uint4*>(o + tile_off<VROWB>(row, p));
        }
    };

    // S^T in units of 1 / sig: S[nj][0, 1] value column col0 + g, keys 8 nj + 2 t, + 1;  S[nj][2, 3] column + 8.  top: a bound of the
    // largest |S| of the row in these units, kept between 2^9 and 2^15 so that the pieces lose nothing at either end of fp16.
    float S[NJ][4], sig[2], inv[2], top[2];
    {
        const float* src = a.states + ((in < 0 ? 0 : in) * a.HV + head) * (long long)(DK * a.DV) + col0 + g;
#pragma unroll
        for (int nj = 0; nj < NJ; ++nj)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[nj][e] = in < 0 ? 0.0f : src[(8 * nj + 2 * t + (e & 1)) * (long long)a.DV + 8 * (e >> 1)];
    }
    last_is_done();
#pragma unroll
    for (int c = 0; c < NSLOT - 1; ++c) issue(c);
    if (NB == 0) {                                               // nothing to walk: the state as it is
        cp_wait<0>();
        float* dst = a.states + (out * a.HV + head) * (long long)(DK * a.DV) + col0 + g;
#pragma unroll
        for (int nj = 0; nj < NJ; ++nj)
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[(8 * nj + 2 * t + (e & 1)) * (long long)a.DV + 8 * (e >> 1)] = S[nj][e];
        return;
    }
    auto row_top = [&](int h) {                                  // the row's largest |S|
        float m = 0.0f;
#pragma unroll
        for (int nj = 0; nj < NJ; ++nj) m = fmaxf(m, fmaxf(fabsf(S[nj][2 * h]), fabsf(S[nj][2 * h + 1])));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        return fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float m = row_top(h);
        const int b = m > 0.0f ? clampi(265 - exponent_of(m), 27, 191) : 127;        // m sig in [2^11, 2^12)
        sig[h] = pow2_biased(b);
        inv[h] = pow2_biased(254 - b);
        top[h] = m * sig[h];
#pragma unroll
        for (int nj = 0; nj < NJ; ++nj) { S[nj][2 * h] *= sig[h]; S[nj][2 * h + 1] *= sig[h]; }
    }
    cp_wait<NSLOT - 2>();
    __syncthreads();
    convert(0);

    for (int c = 0; c < NB; ++c) {
        cp_wait<NSLOT - 3>();                                    // this thread's copies of chunk c + 1 have landed
        __syncthreads();                                         // everyone's; chunk c is converted; chunk c - 1's slot is free
        issue(c + NSLOT - 1);
        convert(c + 1);
        if (c > 0) store_rows(c - 1);
        const Stage<DK, VC>& st = sm.st[c % NSLOT];
        const uint32_t k_s = smem_u32(st.k), q_s = smem_u32(st.q);
        auto wf = [&](int at, int i) { return *reinterpret_cast<const float2*>(st.w + at + i * 4); };
        // ---------------------------------------------------------------- (K S0)^T and (Q S0)^T
        float R[2][4] = {}, RL[2][4] = {}, QS[2][4] = {};
#pragma unroll
        for (int p = 0; p < KSTEP; ++p) {
            const uint32_t off = tile_off<ROWB>((lm >> 1) * 8 + lr, 2 * p + (lm & 1));
            uint32_t bk[4], bq[4], sh[4], sl[4];
            ldsm4(k_s + off, bk);
            ldsm4(q_s + off, bq);
            split_pair(S[2 * p][0], S[2 * p][1], sh[0], sl[0]);
            split_pair(S[2 * p][2], S[2 * p][3], sh[1], sl[1]);
            split_pair(S[2 * p + 1][0], S[2 * p + 1][1], sh[2], sl[2]);
            split_pair(S[2 * p + 1][2], S[2 * p + 1][3], sh[3], sl[3]);
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) {
                mma16<__half>(R[ni], sh, bk[2 * ni], bk[2 * ni + 1]);
                mma16<__half>(RL[ni], sl, bk[2 * ni], bk[2 * ni + 1]);
                mma16<__half>(QS[ni], sh, bq[2 * ni], bq[2 * ni + 1]);
                mma16<__half>(QS[ni], sl, bq[2 * ni], bq[2 * ni + 1]);
            }
        }
        // ---------------------------------------------------------------- W = V - e K S0, scaled by row to at most 2^10; U = T W
        uint32_t vv[4];
        {
            const int p = warp * 2 + (lm & 1);
            ldsm4t(smem_u32(st.v) + tile_off<VROWB>((lm >> 1) * 8 + lr, p), vv);
        }
        // vv[0]: column g, tokens 2t, + 1 | vv[1]: column g + 8 | vv[2], vv[3]: tokens 8 + 2t, + 1
        float Wt[2][4];
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            const float2 er = wf(PW_ER, 8 * ni + 2 * t);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const T* two = reinterpret_cast<const T*>(&vv[2 * ni + h]);
                Wt[ni][2 * h] = fmaf(-er.x, R[ni][2 * h] + RL[ni][2 * h], to_float(two[0]) * sig[h]);
                Wt[ni][2 * h + 1] = fmaf(-er.y, R[ni][2 * h + 1] + RL[ni][2 * h + 1], to_float(two[1]) * sig[h]);
            }
        }
        float uf[2], U[2][4];
        const float tau = *reinterpret_cast<const float*>(st.w + PW_TAU);
        const uint32_t toff = uint32_t(((lm >> 1) * 8 + lr) * 32 + (lm & 1) * 16);
        auto solve = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float m = fmaxf(fmaxf(fabsf(Wt[0][2 * h]), fabsf(Wt[0][2 * h + 1])), fmaxf(fabsf(Wt[1][2 * h]), fabsf(Wt[1][2 * h + 1])));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const int b = clampi(exponent_of(m), 27, 227);
                const float sc = pow2_biased(263 - b);           // m sc in [2^9, 2^10)
                uf[h] = pow2_biased(b - 9) * tau;
#pragma unroll
                for (int ni = 0; ni < 2; ++ni) { Wt[ni][2 * h] *= sc; Wt[ni][2 * h + 1] *= sc; }
            }
            uint32_t wh[4], wl[4], bt[4], btl[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split_pair(Wt[i >> 1][2 * (i & 1)], Wt[i >> 1][2 * (i & 1) + 1], wh[i], wl[i]);
            ldsm4(smem_u32(st.w + PW_T) + toff, bt);
            ldsm4(smem_u32(st.w + PW_TL) + toff, btl);
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) {
                float hi[4] = {}, lo[4] = {};
                mma16<__half>(hi, wh, bt[2 * ni], bt[2 * ni + 1]);
                mma16<__half>(lo, wl, bt[2 * ni], bt[2 * ni + 1]);
                mma16<__half>(lo, wh, btl[2 * ni], btl[2 * ni + 1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) U[ni][e] = hi[e] + lo[e];
            }
        };
        solve();
        // What is no number, or none any more, belongs to its own token and those behind it, but a product's zeros in front of it spread
        // it over the whole chunk.  Such a column is solved again with zeros from there on, and marked from there on.
        const float sound = 0.0f * (((U[0][0] + U[0][1]) + (U[0][2] + U[0][3])) + ((U[1][0] + U[1][1]) + (U[1][2] + U[1][3])));
        const bool unsound = __any_sync(0xffffffffu, sound != 0.0f);
        int first[2] = {PB, PB};
        if (unsound) {
            auto cut = [&](float (&x)[2][4]) {                   // zeros from the first bad token of a column on
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int i = 3; i >= 0; --i) {
                        const int tok = 8 * (i >> 1) + 2 * t + (i & 1);
                        if (!(fabsf(x[i >> 1][2 * h + (i & 1)]) <= 3.402823466e38f)) first[h] = min(first[h], tok);
                    }
                    first[h] = min(first[h], __shfl_xor_sync(0xffffffffu, first[h], 1));
                    first[h] = min(first[h], __shfl_xor_sync(0xffffffffu, first[h], 2));
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (8 * (i >> 1) + 2 * t + (i & 1) >= first[h]) x[i >> 1][2 * h + (i & 1)] = 0.0f;
                }
            };
            const float w0 = uf[0] / tau, w1 = uf[1] / tau;       // W as it was, to be scaled anew
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) { Wt[ni][0] *= w0; Wt[ni][1] *= w0; Wt[ni][2] *= w1; Wt[ni][3] *= w1; }
            cut(Wt);
            solve();
            cut(U);
        }
        const float nan = __int_as_float(0x7fffffff);
        // ---------------------------------------------------------------- what the state takes: D = exp(c_16 - c_j) U, in its units
        float D[2][4], sum[2] = {0.0f, 0.0f}, f[2] = {1.0f, 1.0f};
        const float e16 = *reinterpret_cast<const float*>(st.w + PW_E16);
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
            const float2 dk = wf(PW_DK, 8 * ni + 2 * t);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                D[ni][2 * h] = U[ni][2 * h] * (uf[h] * dk.x);
                D[ni][2 * h + 1] = U[ni][2 * h + 1] * (uf[h] * dk.y);
                if (unsound && first[h] < PB) D[ni][2 * h] = D[ni][2 * h + 1] = nan;
                sum[h] += fabsf(D[ni][2 * h]) + fabsf(D[ni][2 * h + 1]);
            }
        }
        bool far = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
            top[h] = fmaf(e16, top[h], sum[h]);                  // |k| < 1 in its units
            far |= !(top[h] <= 32768.0f && (top[h] >= 512.0f || top[h] == 0.0f));
        }
        // ---------------------------------------------------------------- O = M U + e Q S0
        {
            uint32_t uh[4], ul[4], bm[4], bml[4], ov[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split_pair(U[i >> 1][2 * (i & 1)], U[i >> 1][2 * (i & 1) + 1], uh[i], ul[i]);
            ldsm4(smem_u32(st.w + PW_M) + toff, bm);
            ldsm4(smem_u32(st.w + PW_ML) + toff, bml);
#pragma unroll
            for (int ni = 0; ni < 2; ++ni) {
                float acc[4] = {};
                mma16<__half>(acc, uh, bm[2 * ni], bm[2 * ni + 1]);
                mma16<__half>(acc, ul, bm[2 * ni], bm[2 * ni + 1]);
                mma16<__half>(acc, uh, bml[2 * ni], bml[2 * ni + 1]);
                const float2 om = wf(PW_OM, 8 * ni + 2 * t), eq = wf(PW_EQ, 8 * ni + 2 * t);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = inv[h] * fmaf(acc[2 * h] * uf[h], om.x, eq.x * QS[ni][2 * h]);
                    float y = inv[h] * fmaf(acc[2 * h + 1] * uf[h], om.y, eq.y * QS[ni][2 * h + 1]);
                    if (unsound) {
                        if (8 * ni + 2 * t >= first[h]) x = nan;
                        if (8 * ni + 2 * t + 1 >= first[h]) y = nan;
                    }
                    T two[2] = {from_float<T>(x), from_float<T>(y)};
                    ov[2 * ni + h] = *reinterpret_cast<uint32_t*>(two);
                }
            }
            // matrices (tokens 8 (m / 2) .., columns 8 (m % 2) ..), transposed on the way
            stsm4t(smem_u32(sm.o[c & 1]) + tile_off<VROWB>((lm >> 1) * 8 + lr, warp * 2 + (lm & 1)), ov);
        }
        // ---------------------------------------------------------------- S = e_16 S0 + K^T D
        if (__any_sync(0xffffffffu, far)) {                      // the bound has left its range: the true one, and a scale for it
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = fmaf(e16, row_top(h), sum[h]);
                const int b = exponent_of(sig[h]);
                const int nb = top[h] > 0.0f ? clampi(b + clampi(138 - exponent_of(top[h]), -100, 100), 27, 191) : b;     // top in [2^11, 2^12)
                f[h] = pow2_biased(127 + clampi(nb - b, -120, 120));
                top[h] *= f[h];
            }
        }
        uint32_t dh[4], dl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_pair(D[i >> 1][2 * (i & 1)] * f[i & 1], D[i >> 1][2 * (i & 1) + 1] * f[i & 1], dh[i], dl[i]);
        const float2 ef0 = make_float2(e16 * f[0], e16 * f[0]), ef1 = make_float2(e16 * f[1], e16 * f[1]);
#pragma unroll
        for (int q = 0; q < KSTEP; ++q) {
            uint32_t kf[4];                                      // kf[2 h + c]: keys 16 q + 8 h + g, tokens 8 c + 2 t, + 1
            ldsm4t(k_s + tile_off<ROWB>((lm & 1) * 8 + lr, 2 * q + (lm >> 1)), kf);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float P[4] = {};
                mma16<__half>(P, dh, kf[2 * h], kf[2 * h + 1]);
                mma16<__half>(P, dl, kf[2 * h], kf[2 * h + 1]);
                float (&s)[4] = S[2 * q + h];
                const float2 lo = fma2(ef0, make_float2(s[0], s[1]), make_float2(P[0], P[1]));
                const float2 hi = fma2(ef1, make_float2(s[2], s[3]), make_float2(P[2], P[3]));
                s[0] = lo.x; s[1] = lo.y; s[2] = hi.x; s[3] = hi.y;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sig[h] *= f[h];
            inv[h] = pow2_biased(254 - exponent_of(sig[h]));
        }
    }
    cp_wait<0>();
    __syncthreads();
    store_rows(NB - 1);
    if (out >= 0) {
        float* dst = a.states + (out * a.HV + head) * (long long)(DK * a.DV) + col0 + g;
#pragma unroll
        for (int nj = 0; nj < NJ; ++nj)
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[(8 * nj + 2 * t + (e & 1)) * (long long)a.DV + 8 * (e >> 1)] = S[nj][e] * inv[e >> 1];
    }
}

template <typename T, int DK, int NW, int NSLOT> int launch_scan(const shvk_gdn_seq_args& a, const uint8_t* ws, cudaStream_t s) {
    constexpr int smem = int(sizeof(ScanSmem<DK, 16 * NW, NSLOT>));
    const long long ctas = (long long)a.n_seq * a.HV * (a.DV / (16 * NW));
    if (ctas > 0x7fffffff) return int(cudaErrorInvalidValue);
    const cudaError_t e = cudaFuncSetAttribute(gdn_prefill_scan_kernel<T, DK, NW, NSLOT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return int(e);
    if (a.n_tokens > 0) return int(launch_behind(gdn_prefill_scan_kernel<T, DK, NW, NSLOT>, ctas, NW * 32, smem, s, a, ws));
    gdn_prefill_scan_kernel<T, DK, NW, NSLOT><<<unsigned(ctas), NW * 32, smem, s>>>(a, ws);      // (behind no preparation)
    return int(cudaGetLastError());
}

// Whether the chunks of 64 tokens take a call: sequences that on average fill two.  us, 64 / 16, bf16, 6 heads: DK 128, 128 sequences of 48
// tokens 130 / 80, 64 101 / 99, 72 162 / 113, 112 171 / 147, 128 143 / 160, of none to 256 184 / 187; 512 of 64 345 / 360, of 96 584 / 489, of
// 128 492 / 606, of 321 1,140 / 1,418; 37 of 500 136 / 171.  DK 64: 128 of 64 81 / 58, of 128 114 / 102; 37 of 500 111 / 120; 1 of 1,000 65 / 79.
// Heads that leave half of the 128 lanes idle go there while one wave of CTAs holds them, from two chunks on (DV 64, DK 64, 8 of 256 29 / 27,
// of 2,048 133 / 205, but 37 of 256 58 / 38; DK 128, 1 of 128 21 / 24), and with the wider keys from eight chunks on (128 of 256 210 / 198, of
// 512 357 / 378; 64 of 2,048 625 / 746; DK 64 537 / 441).
inline bool takes_tc(const shvk_gdn_seq_args& a) {
    auto at_least = [&](long long tokens) { return a.n_tokens >= a.n_seq * tokens; };
    if (a.DV % 128 == 0) return at_least(128);
    if (a.DV % 64) return false;
    return (at_least(128) && (long long)a.n_seq * a.HV * ((a.DV + 127) / 128) <= device_sms()) || (a.DK == 128 && at_least(512));
}

inline long long prefill_chunks(const shvk_gdn_seq_args& a) { return a.n_tokens / PB + a.n_seq + 1; }

template <typename T, int DK> int launch_prefill(const shvk_gdn_seq_args& a, uint8_t* ws, cudaStream_t s) {
    const long long items = prefill_chunks(a) * a.HV, ctas = (items + 7) / 8;
    if (ctas > 0x7fffffff) return int(cudaErrorInvalidValue);
    if (a.n_tokens > 0) {
        constexpr int smem = 4 * int(sizeof(PrepWarp<DK>));
        const cudaError_t e = cudaFuncSetAttribute(gdn_prefill_prep_kernel<T, DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return int(e);
        if (const cudaError_t le = launch_behind(gdn_prefill_prep_kernel<T, DK>, ctas, 128, smem, s, a, ws, items); le != cudaSuccess) return int(le);
    }
    // Four warps wherever they divide the columns.  us with two, four and eight warps a CTA, DV 128, sequences of 48 tokens, 6 heads: DK 128, 8 of
    // them 19.0, 17.9, -; 50 41.3, 38.3, 41.0; 128 82.8, 79.5, 84.7; DK 64, 128 50.3, 48.4, 52.9 (two CTAs of four warps and 220 registers stand
    // on an SM, one of eight; two warps bring K and Q in twice as often).
    return a.DV % 64 == 0 ? launch_scan<T, DK, 4, 4>(a, ws, s) : launch_scan<T, DK, 2, 4>(a, ws, s);
}

}  // namespace
}  // namespace sb

extern "C" size_t shvk_gdn_prefill_workspace_bytes(const shvk_gdn_seq_args* a) {
    using namespace sb;
    if (check_gdn_seq(a) || a->n_seq == 0 || a->dtype == DT_F32) return 0;
    if (takes_tc(*a)) return gdn_prefill_tc_workspace(*a);
    return size_t(prefill_chunks(*a)) * size_t(a->HV) * size_t(PW_BYTES);
}

namespace {
int prefill(const shvk_gdn_seq_args* a, void* workspace, size_t workspace_bytes, void* stream, int starve_polls) {
    using namespace sb;
    if (const int e = check_gdn_seq(a)) return e;
    if (a->dtype == DT_F32) return int(cudaErrorInvalidValue);
    if (a->n_seq == 0) return 0;
    if (!workspace || !aligned16(workspace) || workspace_bytes < shvk_gdn_prefill_workspace_bytes(a)) return int(cudaErrorInvalidValue);
    cudaStream_t s = cudaStream_t(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (takes_tc(*a)) return gdn_prefill_tc(*a, ws, s, starve_polls);
    if (starve_polls) return int(cudaErrorInvalidValue);         // the other form waits for nothing that could stay away
    if (a->dtype == DT_BF16) return a->DK == 64 ? launch_prefill<__nv_bfloat16, 64>(*a, ws, s) : launch_prefill<__nv_bfloat16, 128>(*a, ws, s);
    return a->DK == 64 ? launch_prefill<__half, 64>(*a, ws, s) : launch_prefill<__half, 128>(*a, ws, s);
}
}  // namespace

extern "C" int shvk_gdn_prefill(const shvk_gdn_seq_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    return prefill(a, workspace, workspace_bytes, stream, 0);
}

extern "C" int shvk_gdn_prefill_starved(const shvk_gdn_seq_args* a, void* workspace, size_t workspace_bytes, int polls, void* stream) {
    return prefill(a, workspace, workspace_bytes, stream, polls > 1 ? polls : 1);
}
