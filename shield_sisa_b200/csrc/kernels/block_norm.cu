// What stands between two blocks of a layer, in one pass over the rows:
//
//   y = x;  y = y rstd(y) post_w;  y = y act(gate);  h = h_in + scale y;  h_out = h;  xn = h rstd(h) pre_w
// with rstd(z) = 1 / sqrt(mean(z^2) + eps), every step in float32 and each output rounded once.  HBM binds: a row's arrays are read
// once into registers, its two sums of squares are reductions over the threads that hold the row.
//
// A thread has NV groups of eight consecutive values (16-byte accesses): 8 or 16 threads, a warp or a whole CTA to a row, by its length.
// Rows whose pitch is no multiple of eight start anywhere in such a group.  All arrays of a call then start at the same place of it (or
// the call goes to block_norm_any_kernel), and the place repeats every eight rows at most: a CTA walks rows of one class, which are
// cut at the same places, so that its copy of the weights in shared memory, shifted as its rows are, serves them all with 16-byte
// reads.  A group that reaches over a row's end is read whole where that stays in the array, and written value by value.
//
// 16-bit rows, one B200: 123,264 heads of 128 with a SiLU gate 20.2 us (95 MB, 0.71 of a plain copy's rate), 20,544 x 384 residual and norm
// 18.2 us (0.79), four times as many rows of either 5.4 and 6.1 TB/s (0.82, 0.93): ramp up and drain.  16,384 x 2,048 with everything
// 65 us (4.1 TB/s; two barriers of a CTA a row), x 2,047 93: masks at a row's ends, and sectors that two SMs write.
#include "block_norm_rows.cuh"
#include "device_utils.cuh"
#include "launch_order.cuh"
#include "shv_seq_kernels.h"

#include <type_traits>

namespace sb {
namespace {

constexpr int BN_MAXD = 16384;

template <typename T> __device__ __forceinline__ void get8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
    }
}
template <typename T> __device__ __forceinline__ void put8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 w;
        T* e = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = w;
    }
}

// A group of eight values as it lies in memory: 16 or 32 bytes.
template <typename T> struct Raw { uint4 w[sizeof(T) == 4 ? 2 : 1]; };
// The values [lo, hi) of a group, the others as it may be: the whole group in one or two accesses where all of it lies in the array
// (`whole`: everywhere but at an array's end), else value by value.  (Value by value at every row's edges, loads waited for one another:
// 189 us for 16,384 rows of 2,047, now 93.)
template <typename T> __device__ __forceinline__ Raw<T> get_raw(const T* p, int lo, int hi, bool whole) {
    Raw<T> r;
    if (whole) {
#pragma unroll
        for (int i = 0; i < int(sizeof(r.w) / 16); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[min(max(i, lo), hi - 1)];
    }
    return r;
}
template <typename T> __device__ __forceinline__ void values_of(const Raw<T>& r, int lo, int hi, float (&v)[8]) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
    if (hi - lo != 8)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < lo || i >= hi) v[i] = 0.0f;
}

// sigmoid(g) for outputs in TH.  What a gate of -90 leaves of a large value is not nothing, so exp(-g) must not overflow: it is taken of
// -|g|, or 2^-64 times as large.  16-bit outputs: the hardware's exponential and reciprocal, off by the rounding of the exponent, 2^-17 at
// most (a hundredth of half a step of bf16, a thirtieth of fp16's).  float32 outputs: the exponential's argument is a product whose
// rounding error an FMA gives exactly, the reciprocal gets one step of Newton's iteration; some 2^-21 off.  (With expf and a division, 20,544
// rows of 384 with a gate took 26.6 us.)
template <typename TH> __device__ __forceinline__ float sigmoid_of(float g) {
    constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.92596299e-8f, LN2 = 0.693147181f;
    float e, r;
    if constexpr (sizeof(TH) == 4) {
        float x = fabsf(g);
        x = x > 200.0f ? 200.0f : x;                             // (exp(-200) is 0; what is no number stays)
        const float t = x * LOG2E, rest = fmaf(x, LOG2E_REST, fmaf(x, LOG2E, -t));
        asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(-t));
        e = fmaf(e, -LN2 * rest, e);
        const float d = 1.0f + e;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
        r = fmaf(fmaf(-d, r, 1.0f), r, r);
        return g < 0.0f ? e * r : r;
    } else {
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g, -LOG2E, -64.0f)));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0x1p-64f + e));
        return 0x1p-64f * r;
    }
}
template <typename TH> __device__ __forceinline__ float gate_of(float g, int act) {
    return act == 0 ? g : act == 1 ? g * sigmoid_of<TH>(g) : sigmoid_of<TH>(g);
}
// x *= act(g)
template <typename TH> __device__ __forceinline__ void gate8(float (&x)[8], const float (&g)[8], int act) {
    if (act == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= g[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= (act == 1 ? g[e] : 1.0f) * sigmoid_of<TH>(g[e]);
    }
}

// ROWT: threads of a row: 8, 16, 32, or 0 = the whole CTA.  EDGE: a group may reach over a row's ends.  P: classes of rows (1 where every row
// starts on a group).  The next row's values are asked for before this one's are used (not with four groups a thread: no registers).
template <typename T, typename TH, int NV, int ROWT, bool EDGE>
__global__ void __launch_bounds__(ROWT ? 128 : 512, ROWT ? 4 : NV == 1 ? 2 : 1)
block_norm_kernel(const shvk_block_norm_args a, int P) {
    extern __shared__ __align__(16) float bn_w[];                // post_w | pre_w | gate row, each `span` floats
    __shared__ __align__(16) float red[2][2][16];                            // [row parity][which sum][warp]
    const int tid = threadIdx.x, rt = ROWT ? ROWT : blockDim.x, span = rt * NV * 8;
    const int groups = ROWT ? blockDim.x / ROWT : 1, grp = ROWT ? tid / ROWT : 0, j = ROWT ? tid % ROWT : tid;
    const int cls = blockIdx.x % P, cta = blockIdx.x / P, total = int(a.rows * a.heads);
    const int off = row_shift(cls, a.ldx);                       // where the class's rows start in a group (0 where P is 1)
    // this group's rows are R, R + step, ...; as (row, head) they move by (step_row, step_head)
    const int step = int(gridDim.x / P) * groups * P, step_row = step / a.heads, step_head = step % a.heads;
    int R = (cta * groups + grp) * P + cls, row = R / a.heads, head = R % a.heads;
    const bool post = a.post_w, pre = a.pre_w, one_gate = a.gate && a.ldgate == 0 && a.heads == 1, row_gate = a.gate && !one_gate;
    const float inv_d = 1.0f / float(a.D);
    const int width = a.heads * a.D;                             // of a row
    int lo[NV], hi[NV];                                          // the values of each group that belong to the row: [lo, hi)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (j + i * rt) * 8 - off;                    // column of the group's first value
        lo[i] = EDGE ? group_lo(c) : 0;
        hi[i] = EDGE ? group_hi(c, a.D) : c < a.D ? 8 : 0;
    }
    int whole = 0;                                               // rows in which a group over the row's end is read whole
    if (EDGE) {
        whole = whole_rows(int(a.rows), a.ldx);
        if (a.h_in) whole = min(whole, whole_rows(int(a.rows), a.ldh_in));
        if (row_gate) whole = min(whole, whole_rows(int(a.rows), a.ldgate));
    }
    auto full = [&](int i) { return !EDGE || hi[i] - lo[i] == 8; };
    struct Row {
        Raw<T> x[NV], g[NV];
        Raw<TH> h[NV];
    };
    // the values of (row, head); where there are none (no such row, no such group) zeros
    auto fetch = [&](bool on, int row, int head, Row& r) {
        const uint4 z = make_uint4(0, 0, 0, 0);
        const int base = head * a.D - off + j * 8;
        const T* px = static_cast<const T*>(a.x) + row * a.ldx + base;
        const T* pg = static_cast<const T*>(a.gate) + row * a.ldgate + base;
        const TH* ph = static_cast<const TH*>(a.h_in) + row * a.ldh_in + base;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            r.x[i].w[0] = r.g[i].w[0] = z;
            r.h[i].w[0] = z;
            if constexpr (sizeof(T) == 4) r.x[i].w[1] = r.g[i].w[1] = z;
            if constexpr (sizeof(TH) == 4) r.h[i].w[1] = z;
            if (on && hi[i] > lo[i]) {
                const int c = i * rt * 8;
                const bool all = !EDGE || reads_whole(base + c + 8, width, row, whole);
                r.x[i] = get_raw(px + c, lo[i], hi[i], all);
                if (a.h_in) r.h[i] = get_raw(ph + c, lo[i], hi[i], all);
                if (row_gate) r.g[i] = get_raw(pg + c, lo[i], hi[i], all);
            }
        }
    };
    auto store = [&](auto* p, int i, const float (&v)[8]) {
        if (full(i)) {
            put8(p, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= lo[i] && e < hi[i]) p[e] = from_float<std::remove_pointer_t<decltype(p)>>(v[e]);
        }
    };
    constexpr bool AHEAD = NV < 4;
    Row now;
    next_may_start();
    last_is_done();
    fetch(R < total, row, head, now);
    if (ROWT == 0 && tid < 64) (&red[0][0][0])[tid] = 0.0f;
    for (int e = tid; e < span; e += blockDim.x) {               // the weights, behind the first row's loads
        const int c = e - off;
        const bool in = c >= 0 && c < a.D;
        if (post) bn_w[e] = in ? a.post_w[c] : 0.0f;
        if (pre) bn_w[span + e] = in ? a.pre_w[c] : 0.0f;
        if (one_gate) bn_w[2 * span + e] = in ? gate_of<TH>(to_float(static_cast<const T*>(a.gate)[c]), a.gate_act) : 0.0f;
    }
    __syncthreads();
    int par = 0;
    // whole CTAs walk the rows in step: a group without a row of its own goes along without touching memory
    for (int first = cta * groups * P + cls; first < total; first += step, par ^= 1) {
        const bool on = R < total;
        const int this_row = row, this_base = head * a.D - off + j * 8;
        R += step;
        row += step_row;
        head += step_head;
        if (head >= a.heads) {
            head -= a.heads;
            ++row;
        }
        Row next;
        if (AHEAD) fetch(R < total, row, head, next);
        float x[NV][8], h[NV][8], ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float gt[8];
            values_of(now.x[i], EDGE ? lo[i] : 0, EDGE ? hi[i] : 8, x[i]);
            values_of(now.h[i], EDGE ? lo[i] : 0, EDGE ? hi[i] : 8, h[i]);
            if (row_gate) values_of(now.g[i], EDGE ? lo[i] : 0, EDGE ? hi[i] : 8, gt);
            if (post)
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(x[i][e], x[i][e], ss);
            if (row_gate)                                        // the row's rstd is one factor of all its values: the gate may go first
                gate8<TH>(x[i], gt, a.gate_act);
        }
        auto row_sum = [&](float v, int which) {
#pragma unroll
            for (int o = ROWT ? ROWT / 2 : 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if constexpr (ROWT == 0) {
                if ((tid & 31) == 0) red[par][which][tid >> 5] = v;
                __syncthreads();
                v = 0.0f;
#pragma unroll
                for (int w = 0; w < 16; w += 4)                  // (no more than sixteen warps, the sums of those that are not there zero)
                    if (w * 32 < blockDim.x) {
                        const float4 q = *reinterpret_cast<const float4*>(&red[par][which][w]);
                        v += (q.x + q.y) + (q.z + q.w);
                    }
            }
            return v;
        };
        if (post) {
            const float r = rsqrtf(row_sum(ss, 0) * inv_d + a.eps);      // (two steps of 2^-23 off at most)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float w[8];
                get8<float>(bn_w + (j + i * rt) * 8, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = x[i][e] * r * w[e];
            }
        }
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (one_gate) {
                float w[8];
                get8<float>(bn_w + 2 * span + (j + i * rt) * 8, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] *= w[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i][e] = fmaf(x[i][e], a.scale, h[i][e]);       // (h is zero where there is no residual)
            if (pre)
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
            if (on && hi[i] > lo[i] && a.h_out) store(static_cast<TH*>(a.h_out) + this_row * a.ldh_out + this_base + i * rt * 8, i, h[i]);
        }
        if (pre) {
            const float r = rsqrtf(row_sum(ss, 1) * inv_d + a.eps);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float w[8];
                get8<float>(bn_w + span + (j + i * rt) * 8, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = h[i][e] * r * w[e];
                if (on && hi[i] > lo[i]) store(static_cast<T*>(a.xn) + this_row * a.ldxn + this_base + i * rt * 8, i, w);
            }
        }
        if (AHEAD) now = next;
        else fetch(R < total, row, head, now);
    }
}

// Any pitch and alignment: a CTA per row, value by value, the row's h in shared memory (h_out may be h_in, so h is not made twice).
template <typename T, typename TH>
__global__ void __launch_bounds__(256) block_norm_any_kernel(const shvk_block_norm_args a) {
    extern __shared__ float bn_h[];
    __shared__ float red[2][8];
    const int tid = threadIdx.x;
    next_may_start();
    last_is_done();
    const long long row = blockIdx.x / a.heads, base = blockIdx.x % a.heads * (long long)a.D;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx + base;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + row * a.ldgate + base : nullptr;
    const TH* h_in = a.h_in ? static_cast<const TH*>(a.h_in) + row * a.ldh_in + base : nullptr;
    auto row_sum = [&](float v, int which) {
        v = warp_sum(v);
        if ((tid & 31) == 0) red[which][tid >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += red[which][w];
        return v;
    };
    float r = 1.0f, ss = 0.0f;
    if (a.post_w) {
        for (int c = tid; c < a.D; c += 256) {
            const float v = to_float(x[c]);
            ss = fmaf(v, v, ss);
        }
        r = 1.0f / sqrtf(row_sum(ss, 0) / float(a.D) + a.eps);
    }
    ss = 0.0f;
    for (int c = tid; c < a.D; c += 256) {
        float v = to_float(x[c]);
        if (a.post_w) v = v * r * a.post_w[c];
        if (gate) v *= gate_of<TH>(to_float(gate[c]), a.gate_act);
        v = h_in ? fmaf(v, a.scale, to_float(h_in[c])) : v * a.scale;
        if (a.h_out) static_cast<TH*>(a.h_out)[row * a.ldh_out + base + c] = from_float<TH>(v);
        ss = fmaf(v, v, ss);
        bn_h[c] = v;                                             // read back by this thread alone
    }
    if (a.pre_w) {
        r = 1.0f / sqrtf(row_sum(ss, 1) / float(a.D) + a.eps);
        for (int c = tid; c < a.D; c += 256) static_cast<T*>(a.xn)[row * a.ldxn + base + c] = from_float<T>(bn_h[c] * r * a.pre_w[c]);
    }
}

template <typename T, typename TH, int NV, int ROWT, bool EDGE>
int launch_rows(const shvk_block_norm_args& a, int P, int threads, cudaStream_t s) {
    const int groups = ROWT ? threads / ROWT : 1, span = (ROWT ? ROWT : threads) * NV * 8;
    const int smem = 3 * span * int(sizeof(float));
    // (the kernel's limit is one for all callers: always the most that any of them needs, so that none lowers it under another's launch)
    constexpr int most_smem = 3 * (ROWT ? ROWT : 512) * NV * 8 * int(sizeof(float));
    static_assert(most_smem <= 200 * 1024, "the longest row's weights fit");
    if (smem > 47 * 1024) {                                      // (beside the sums of a CTA, which are static)
        const cudaError_t e = cudaFuncSetAttribute(block_norm_kernel<T, TH, NV, ROWT, EDGE>, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem);
        if (e != cudaSuccess) return int(e);
    }
    const long long need = ((a.rows * a.heads + P - 1) / P + groups - 1) / groups * P;     // CTAs of one pass over the rows
    const int resident = ROWT ? 4 : NV == 1 ? 1024 / threads : threads > 256 ? 1 : 512 / threads;      // CTAs of an SM, by registers
    const long long most = (long long)device_sms() * resident / P * P;
    const long long ctas = need < most ? need : (most > 0 ? most : P);
    return int(launch_behind(block_norm_kernel<T, TH, NV, ROWT, EDGE>, ctas, threads, smem, s, a, P));
}

template <typename T, typename TH, bool EDGE> int launch_vec(const shvk_block_norm_args& a, int P, int nvec, cudaStream_t s) {
    if (nvec <= 16) return launch_rows<T, TH, 2, 8, EDGE>(a, P, 128, s);
    if (nvec <= 32) return launch_rows<T, TH, 2, 16, EDGE>(a, P, 128, s);
    if (nvec <= 64) return launch_rows<T, TH, 2, 32, EDGE>(a, P, 128, s);
    // one group a thread while a CTA may hold the row so (16,384 rows of 2,048: 65 us, two groups 71; of 2,047, with edges: 100 and 93)
    if (!EDGE && nvec <= 512) return launch_rows<T, TH, 1, 0, false>(a, P, (nvec + 31) / 32 * 32, s);
    if (nvec <= 1024) return launch_rows<T, TH, 2, 0, EDGE>(a, P, ((nvec + 1) / 2 + 31) / 32 * 32, s);
    return launch_rows<T, TH, 4, 0, EDGE>(a, P, ((nvec + 3) / 4 + 31) / 32 * 32, s);
}

inline bool on_group(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, typename TH> int launch_block_norm(const shvk_block_norm_args& a, cudaStream_t s) {
    // the vector form: every array starts on 16 bytes, and a row starts at the same place of a group of eight in all of them
    const int ld = int(a.ldx & 7);
    const bool gate_rows = a.gate && (a.ldgate || a.heads > 1);
    const bool vec = on_group(a.x) && on_group(a.h_in) && on_group(a.h_out) && on_group(a.xn) && (!gate_rows || on_group(a.gate)) &&
                     (!a.h_in || (a.ldh_in & 7) == ld) && (!a.h_out || (a.ldh_out & 7) == ld) && (!a.xn || (a.ldxn & 7) == ld) &&
                     (!gate_rows || (a.ldgate & 7) == ld) && (a.heads == 1 || (ld == 0 && a.D % 8 == 0));
    // (by the pitch alone, for one row too: a row's sums are taken in the same order alone and among others)
    const int P = ld == 0 ? 1 : ld % 2 ? 8 : ld % 4 ? 4 : 2, nvec = (a.D + (P > 1 ? 7 : 0) + 7) / 8;
    if (!vec || nvec > 2048) {
        const int smem = a.D * int(sizeof(float));
        const cudaError_t e = cudaFuncSetAttribute(block_norm_any_kernel<T, TH>, cudaFuncAttributeMaxDynamicSharedMemorySize, BN_MAXD * int(sizeof(float)));
        if (e != cudaSuccess) return int(e);
        return int(launch_behind(block_norm_any_kernel<T, TH>, a.rows * a.heads, 256, smem, s, a));
    }
    return P == 1 && a.D % 8 == 0 ? launch_vec<T, TH, false>(a, P, nvec, s) : launch_vec<T, TH, true>(a, P, nvec, s);
}

inline bool on_type(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == DT_F32 ? 3 : 1)) == 0; }

}  // namespace
}  // namespace sb

extern "C" int shvk_block_norm(const shvk_block_norm_args* a, void* stream) {
    using namespace sb;
    constexpr int bad = int(cudaErrorInvalidValue);
    if (!a || a->rows < 0 || a->heads < 1 || a->heads > 4096 || a->D < 1 || a->D > BN_MAXD) return bad;
    const int t = a->x_dtype;
    if (t != DT_F32 && t != DT_BF16 && t != DT_F16) return bad;
    if (a->h_dtype != DT_F32 && a->h_dtype != t) return bad;
    if ((a->gate && (a->gate_dtype != t || a->gate_act < 0 || a->gate_act > 2)) || (a->xn && a->xn_dtype != t)) return bad;
    if (!!a->pre_w != !!a->xn || (!a->h_out && !a->xn)) return bad;
    if (a->rows == 0) return 0;
    if (!a->x) return bad;
    if (a->rows > 0x3fffffff / a->heads) return bad;
    const long long width = (long long)a->heads * a->D;
    if (a->ldx < 0 || (a->h_in && a->ldh_in < 0) || (a->gate && a->ldgate < 0)) return bad;
    if (a->rows > 1 && ((a->h_out && a->ldh_out < width) || (a->xn && a->ldxn < width))) return bad;
    if (!on_type(a->x, t) || !on_type(a->gate, t) || !on_type(a->xn, t) || !on_type(a->h_in, a->h_dtype) || !on_type(a->h_out, a->h_dtype) ||
        !on_type(a->post_w, DT_F32) || !on_type(a->pre_w, DT_F32))
        return bad;
    cudaStream_t s = cudaStream_t(stream);
    shvk_block_norm_args dense = *a;                             // heads that follow one another without a gap are rows
    auto packed = [&](const void* p, long long ld) { return !p || ld == width; };
    if (a->heads > 1 && packed(a->x, a->ldx) && packed(a->gate, a->ldgate) && packed(a->h_in, a->ldh_in) && packed(a->h_out, a->ldh_out) && packed(a->xn, a->ldxn)) {
        dense.rows *= a->heads;
        dense.heads = 1;
        dense.ldx = dense.ldgate = dense.ldh_in = dense.ldh_out = dense.ldxn = a->D;
        a = &dense;
    }
    if (t == DT_F32) return launch_block_norm<float, float>(*a, s);
    if (t == DT_BF16) return a->h_dtype == DT_F32 ? launch_block_norm<__nv_bfloat16, float>(*a, s) : launch_block_norm<__nv_bfloat16, __nv_bfloat16>(*a, s);
    return a->h_dtype == DT_F32 ? launch_block_norm<__half, float>(*a, s) : launch_block_norm<__half, __half>(*a, s);
}
