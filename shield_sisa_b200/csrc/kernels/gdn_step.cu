// The gated delta rule, token by token, with its states in the slots of a pool:
//
//   S <- exp(g) S,  u = beta (v - S^T k),  S <- S + k u^T,  o = S^T q
// in float32, q = scale q / |q| and k = k / |k| where the caller asks for it (|x| = sqrt(x.x + 1e-6)), one key head for HV / HK value
// heads.  Both products with a state are taken before its update, o = exp(g) S^T q + (k.q) u, so that a token costs one sum over the
// keys.  The arithmetic is that of the reference's token loop (engine/cuda/seq.cu:107-195); it has no form that keeps a state.
//
// A token of a sequence moves DK x DV floats in and out for 6 DK DV operations: HBM binds.  A CTA takes VC of a head's value columns, its
// state in registers from the first token to the last: a thread has four columns (16-byte loads and stores) of every RSTEP-th key.
// One token for each of 512 sequences, 6 heads of 128 x 128, bf16: 406 MB in 68 us, 6.0 TB/s, 0.91 of what a plain copy reaches.  (32 value
// columns to a CTA, 128 threads: a CTA asks for 16 KB at once and seven of them are resident, enough bytes in flight; a sequence of several
// tokens pays two barriers of four warps for each.)  128 sequences of float32 values, 6 heads of 64 x 128: 10.5 us, 0.75; below some 50 MB
// the launch and the state's one round trip show.
#include "gdn_seq.cuh"

namespace sb {
namespace {

constexpr int STEP_RPT = 16;                  // keys of a thread's columns: 64 registers of state

// Four consecutive values as float32.
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <typename T> __device__ __forceinline__ float4 load4(const T* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&w);
    return make_float4(to_float(e[0]), to_float(e[1]), to_float(e[2]), to_float(e[3]));
}

template <int DK, int VC> __host__ __device__ constexpr int step_threads() { return DK * (VC / 4) / STEP_RPT; }

template <typename T, int DK, int VC>
__global__ void __launch_bounds__(step_threads<DK, VC>())
gdn_step_kernel(const shvk_gdn_seq_args a) {
    constexpr int NT = step_threads<DK, VC>(), NW = NT / 32, LPR = VC / 4, RSTEP = NT / LPR;
    static_assert(NT % 32 == 0 && 32 % LPR == 0 && RSTEP * STEP_RPT == DK, "whole warps, whole rows");
    __shared__ __align__(16) float qk[2][2][DK];                 // [token parity][q, k]
    __shared__ float dots[2];                                    // k.q of the token
    __shared__ __align__(16) float part[2][NW][2][VC];           // [token parity][warp][S^T k, S^T q]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int splits = a.DV / VC, split = blockIdx.x % splits;
    const int nh = blockIdx.x / splits, n = nh / a.HV, head = nh % a.HV, khead = head / (a.HV / a.HK);
    const int col = split * VC + tid % LPR * 4, row0 = tid / LPR;
    next_may_start();
    last_is_done();
    const SeqRows rows(a.seq_start, n, int(a.n_tokens));
    const long long in = slot_of(a.slot_in, n, a.n_slots), out = slot_of(a.slot_out, n, a.n_slots);
    if (rows.start == rows.end && (out < 0 || out == in)) return;

    float4 S[STEP_RPT];
    if (in >= 0) {
        const float* src = a.states + ((in * a.HV + head) * DK + row0) * a.DV + col;
#pragma unroll
        for (int i = 0; i < STEP_RPT; ++i) S[i] = __ldcs(reinterpret_cast<const float4*>(src + (long long)i * RSTEP * a.DV));
    } else {
#pragma unroll
        for (int i = 0; i < STEP_RPT; ++i) S[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    const T* q = static_cast<const T*>(a.q) + (long long)rows.start * a.ldq + khead * DK;
    const T* k = static_cast<const T*>(a.k) + (long long)rows.start * a.ldk + khead * DK;
    const T* v = static_cast<const T*>(a.v) + (long long)rows.start * a.ldv + (long long)head * a.DV + col;
    T* o = static_cast<T*>(a.o) + (long long)rows.start * a.ldo + (long long)head * a.DV + col;
    const float* g = a.g + (long long)rows.start * a.ldgb + head;
    const float* beta = a.beta + (long long)rows.start * a.ldgb + head;

    for (int t = rows.start, par = 0; t < rows.end; ++t, par ^= 1) {
        if (warp == t % NW) {                                    // one warp prepares q and k; the parity's buffers are two tokens old
            constexpr int E = DK / 32;
            float qe[E], ke[E], qq = 0.0f, kk = 0.0f, kq = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                qe[e] = to_float(q[lane * E + e]);
                ke[e] = to_float(k[lane * E + e]);
                qq = fmaf(qe[e], qe[e], qq);
                kk = fmaf(ke[e], ke[e], kk);
                kq = fmaf(ke[e], qe[e], kq);
            }
            qq = warp_sum(qq);
            kk = warp_sum(kk);
            kq = warp_sum(kq);
            const float rq = a.l2norm ? a.scale / sqrtf(qq + 1e-6f) : a.scale, rk = a.l2norm ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                qk[par][0][lane * E + e] = qe[e] * rq;
                qk[par][1][lane * E + e] = ke[e] * rk;
            }
            if (lane == 0) dots[par] = kq * rq * rk;
        }
        const float4 vv = load4(v);
        const float e = expf(*g), b = *beta;
        __syncthreads();
        float2 r0 = make_float2(0.0f, 0.0f), r1 = r0, s0 = r0, s1 = r0;
#pragma unroll
        for (int i = 0; i < STEP_RPT; ++i) {
            const float kv = qk[par][1][row0 + i * RSTEP], qv = qk[par][0][row0 + i * RSTEP];
            const float2 lo = make_float2(S[i].x, S[i].y), hi = make_float2(S[i].z, S[i].w);
            r0 = fma2(make_float2(kv, kv), lo, r0);
            r1 = fma2(make_float2(kv, kv), hi, r1);
            s0 = fma2(make_float2(qv, qv), lo, s0);
            s1 = fma2(make_float2(qv, qv), hi, s1);
        }
        float4 r = make_float4(r0.x, r0.y, r1.x, r1.y), s = make_float4(s0.x, s0.y, s1.x, s1.y);
#pragma unroll
        for (int off = LPR; off < 32; off <<= 1) {
            r.x += __shfl_xor_sync(0xffffffffu, r.x, off);
            r.y += __shfl_xor_sync(0xffffffffu, r.y, off);
            r.z += __shfl_xor_sync(0xffffffffu, r.z, off);
            r.w += __shfl_xor_sync(0xffffffffu, r.w, off);
            s.x += __shfl_xor_sync(0xffffffffu, s.x, off);
            s.y += __shfl_xor_sync(0xffffffffu, s.y, off);
            s.z += __shfl_xor_sync(0xffffffffu, s.z, off);
            s.w += __shfl_xor_sync(0xffffffffu, s.w, off);
        }
        const int c4 = tid % LPR * 4;
        if (lane < LPR) {
            *reinterpret_cast<float4*>(&part[par][warp][0][c4]) = r;
            *reinterpret_cast<float4*>(&part[par][warp][1][c4]) = s;
        }
        __syncthreads();
        r = s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(&part[par][w][0][c4]), y = *reinterpret_cast<const float4*>(&part[par][w][1][c4]);
            r.x += x.x; r.y += x.y; r.z += x.z; r.w += x.w;
            s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
        }
        const float kq = dots[par];
        const float2 u0 = make_float2(b * (vv.x - e * r.x), b * (vv.y - e * r.y)), u1 = make_float2(b * (vv.z - e * r.z), b * (vv.w - e * r.w));
        if (tid < LPR)
            store_quad<T>(o, fmaf(e, s.x, kq * u0.x), fmaf(e, s.y, kq * u0.y), fmaf(e, s.z, kq * u1.x), fmaf(e, s.w, kq * u1.y));
#pragma unroll
        for (int i = 0; i < STEP_RPT; ++i) {
            const float kv = qk[par][1][row0 + i * RSTEP];
            const float2 lo = fma2(make_float2(e, e), make_float2(S[i].x, S[i].y), mul2(make_float2(kv, kv), u0));
            const float2 hi = fma2(make_float2(e, e), make_float2(S[i].z, S[i].w), mul2(make_float2(kv, kv), u1));
            S[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
        }
        q += a.ldq; k += a.ldk; v += a.ldv; o += a.ldo; g += a.ldgb; beta += a.ldgb;
    }
    if (out >= 0) {
        float* dst = a.states + ((out * a.HV + head) * DK + row0) * a.DV + col;
#pragma unroll
        for (int i = 0; i < STEP_RPT; ++i) __stcs(reinterpret_cast<float4*>(dst + (long long)i * RSTEP * a.DV), S[i]);
    }
}

template <typename T, int DK, int VC> int launch_step(const shvk_gdn_seq_args& a, cudaStream_t s) {
    const long long ctas = (long long)a.n_seq * a.HV * (a.DV / VC);
    if (ctas > 0x7fffffff) return int(cudaErrorInvalidValue);
    return int(launch_behind(gdn_step_kernel<T, DK, VC>, ctas, step_threads<DK, VC>(), 0, s, a));
}

template <typename T> int dispatch_step(const shvk_gdn_seq_args& a, cudaStream_t s) {
    return a.DK == 64 ? launch_step<T, 64, 32>(a, s) : launch_step<T, 128, 32>(a, s);
}

}  // namespace
}  // namespace sb

extern "C" int shvk_gdn_step(const shvk_gdn_seq_args* a, void* stream) {
    using namespace sb;
    if (const int e = check_gdn_seq(a)) return e;
    if (a->n_seq == 0) return 0;
    SB_DISPATCH_DTYPE(a->dtype, T, return dispatch_step<T>(*a, cudaStream_t(stream)))
}
