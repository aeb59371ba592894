// What the two forms of the delta rule with kept states share: the argument checks, and where a packed sequence, its heads and its
// slots lie.
#pragma once
#include "device_utils.cuh"
#include "launch_order.cuh"
#include "shv_seq_kernels.h"

namespace sb {

// The rows [start, end) of sequence n.  Whatever seq_start holds, they lie inside the caller's n_tokens rows.
struct SeqRows {
    int start, end;
    __device__ __forceinline__ SeqRows(const int32_t* __restrict__ seq_start, int n, int n_tokens) {
        start = min(max(seq_start[n], 0), n_tokens);
        end = min(max(seq_start[n + 1], start), n_tokens);
    }
};

// Slot of sequence n, or -1 (no array, or a value that is no slot of the pool).
__device__ __forceinline__ long long slot_of(const int32_t* __restrict__ slots, int n, long long n_slots) {
    const long long s = slots ? slots[n] : -1;
    return s >= 0 && s < n_slots ? s : -1;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// 0, or the error of arguments that no kernel may see.  Rows are read and written in 16-byte pieces.
inline int check_gdn_seq(const shvk_gdn_seq_args* a) {
    constexpr int bad = int(cudaErrorInvalidValue);
    if (!a || a->n_seq < 0 || a->n_tokens < 0 || a->n_tokens > 0x7fffffff) return bad;
    if (a->dtype != DT_F32 && a->dtype != DT_BF16 && a->dtype != DT_F16) return bad;
    if ((a->DK != 64 && a->DK != 128) || a->DV < 32 || a->DV > 256 || a->DV % 32) return bad;
    if (a->HK < 1 || a->HV < 1 || a->HV > 4096 || a->HV % a->HK) return bad;
    if (a->n_seq == 0) return 0;
    if (!a->seq_start || !aligned4(a->seq_start) || !aligned4(a->slot_in) || !aligned4(a->slot_out)) return bad;
    if (a->n_tokens > 0) {
        if (!a->q || !a->k || !a->v || !a->g || !a->beta || !a->o) return bad;
        if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o)) return bad;
        if (!aligned4(a->g) || !aligned4(a->beta)) return bad;
        const long long vec = a->dtype == DT_F32 ? 4 : 8;
        const long long kw = (long long)a->HK * a->DK, vw = (long long)a->HV * a->DV, most = 1ll << 32;
        if (a->ldq < kw || a->ldk < kw || a->ldv < vw || a->ldgb < a->HV || a->ldo < vw) return bad;
        if (a->ldq > most || a->ldk > most || a->ldv > most || a->ldo > most || a->ldgb > most) return bad;
        if ((a->ldq | a->ldk | a->ldv | a->ldo) % vec) return bad;
    }
    if (a->n_slots < 0 || ((a->slot_in || a->slot_out) && (!a->states || !aligned16(a->states)))) return bad;
    return 0;
}

// gdn_prefill_tc.cu: the chunked form for DV a multiple of 64 (arguments checked, tokens there, workspace large enough)
size_t gdn_prefill_tc_workspace(const shvk_gdn_seq_args& a);
int gdn_prefill_tc(const shvk_gdn_seq_args& a, uint8_t* ws, cudaStream_t s, int starve_polls = 0);

}  // namespace sb
