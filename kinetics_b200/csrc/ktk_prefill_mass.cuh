// Interface between the entry point (ktk_prefill_mass.cu) and the tcgen05 kernel (ktk_prefill_mass_umma.cu).
#pragma once

#include "ktk_decode_mma.cuh"

namespace ktk {

struct PrefillMassParams {
    const void* q;
    void* o;                    // fp32
    const void* cache;
    const int32_t* q_indptr;
    const int32_t* kv_indices;
    const int32_t* kv_indptr;
    const int32_t* kv_last_page_len;
    const int32_t* page_count;
    int sink_tokens;
    int batch, Hkv, G;
    int64_t num_pages;
    int64_t total_new;
    int max_new, max_pages;     // the caller's bounds
    float scale_log2;
    void* lse;                  // of the rows [total_new, Hq]: bf16 see prefill_attention (ktk_decode.cuh), fp32 minus log2 of denominators
    int window;
    int32_t* status;
    MassParams m;
    // of the tcgen05 form (mass_plan)
    int splits;                 // parts that the rows of a group of pages are cut into
    float* partial;             // splits > 1: [groups of all sequences][Hkv][splits][256] sums by key
};

// What a CTA's sequence is, and where it lies in the mass array; false: nothing to do
struct MassSequence {
    SeqPages sp;
    int q0, n_new, base_pos, row;
    int counted;                // first new token that counts
};
__device__ __forceinline__ bool mass_sequence(const PrefillMassParams& p, int b, bool first, MassSequence& s) {
    s.q0 = p.q_indptr[b];
    s.n_new = p.q_indptr[b + 1] - s.q0;
    if (s.n_new <= 0) return false;
    s.sp = seq_pages(p.kv_indptr, p.page_count, p.kv_last_page_len, p.sink_tokens, b);
    s.base_pos = s.sp.total - s.n_new;
    s.row = p.m.slot_index ? p.m.slot_index[b] : b;
    s.counted = p.window > 0 && p.window < s.n_new ? s.n_new - p.window : 0;
    if (s.sp.bad || s.base_pos < 0 || s.sp.n_pages > p.max_pages || s.n_new > p.max_new || s.q0 < 0 ||
        s.q0 + (int64_t)s.n_new > p.total_new ||
        s.row < 0 || s.row >= p.m.rows || s.sp.total > p.m.stride) {
        if (first && threadIdx.x == 0) report(p.status, KTK_STATUS_BAD_TABLE);
        return false;
    }
    return true;
}

// How the tcgen05 form cuts its work: groups of 16 pages of all sequences (at most), parts of each, floats of their sums
struct MassPlan {
    int64_t groups;
    int splits;
    size_t partial;
};
MassPlan mass_plan(const ktk_shape* s, int max_new_tokens, int64_t max_pages, int64_t total_pages, int window);
int launch_prefill_mass_f32(const PrefillMassParams& p, cudaStream_t st);      // attention and sums
int launch_prefill_mass_umma(const PrefillMassParams& p, int64_t groups, cudaStream_t st);

}  // namespace ktk
