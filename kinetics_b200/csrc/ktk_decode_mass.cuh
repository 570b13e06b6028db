// Decode attention that adds up weights, one cluster of CTAs per (sequence, kv head): what its kernels do behind the last page.
#pragma once

#include <cooperative_groups.h>

#include "ktk_decode.cuh"

namespace ktk {

constexpr int kMassMaxCluster = 8;
// Pages in flight of a bf16 CTA: 4 with four CTAs per SM; a CTA that has an SM to itself, or shares it with one, needs more to be
// fed.
constexpr int kMassPage = 2 * kPageSize * kHeadDim * 2;
// dynamic shared memory of a bf16 CTA with its share of a list of max_pages
inline int64_t mma_mass_smem(int stages, int max_pages, int cluster, int G) {
    return 1024 + stages * kMassPage + (max_pages + cluster - 1) / cluster * (int64_t)(kPageSize * G * sizeof(float));
}
// bf16 CTAs that an SM holds, beside their static shared memory and what the system takes of it
inline int mma_mass_per_sm(int stages, int max_pages, int cluster, int G) {
    return (int)(228 * 1024 / (mma_mass_smem(stages, max_pages, cluster, G) + 6 * 1024));
}

// A CTA's share of a list: entries [e0, e1)
struct ListShare {
    EntryList el;
    int e0, e1;
};

// What the CTAs of a cluster read of each other
template <int G_MAX> struct MassShared {
    float ml[G_MAX][2];                       // running maximum (log2 domain), sum
    float o[G_MAX][kHeadDim];                 // un-normalised outputs
    float weight[kMassMaxCluster][G_MAX];     // of each CTA's outputs
    float neg_lse[G_MAX];
};

// Behind a barrier of the CTA: `sh` holds its partial result, `scores` [16 (e1 - e0)][G] those of its tokens (log2 domain).  Writes the
// outputs, each CTA of the cluster its part of them, and the masses of the CTA's tokens.  All threads of the cluster.
template <typename T, int G_MAX>
__device__ __forceinline__ void finish_cluster(const DecodeParams& p, const MassParams& m, int b, int h, int G, int cluster, int rank,
                                               MassShared<G_MAX>& sh, const float* scores, const ListShare& share) {
    constexpr int kEach = 4;                  // tokens of a thread, their loads in flight together
    const int tid = threadIdx.x, threads = blockDim.x;
    const EntryList& el = share.el;
    const int tokens = el.cnt == 0 ? 0 : el.cnt == 1 ? el.last : el.first + (el.cnt - 2) * kPageSize + el.last;
    const int row = m.slot_index ? m.slot_index[b] : b;
    const bool on = tokens > 0 && row >= 0 && row < m.rows && tokens <= m.stride;
    if (tokens > 0 && !on && tid == 0 && rank == 0) report(p.status, KTK_STATUS_BAD_TABLE);
    const int64_t at = on ? ((int64_t)row * p.Hkv + h) * m.stride : 0;
    const int n = on ? (share.e1 - share.e0) * kPageSize : 0;
    // token of the i-th place of the share; -1: none there
    const auto token = [&](int i) {
        const int e = share.e0 + i / kPageSize, slot = i % kPageSize;
        return slot < entry_tokens(el, e) ? page_first_pos(e, el.first) + slot : -1;
    };
    float before[kEach];                      // the first ones', on their way across the barrier
    const auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int i = i0 + k * threads + tid, t = i < n ? token(i) : -1;
            before[k] = t >= 0 && t != tokens - 1 ? m.in[at + t] : 0.0f;
        }
    };
    load(0);
    auto cl = cooperative_groups::this_cluster();
    if (cluster > 1) cl.sync();
    const auto theirs = [&](const float* mine, int r) { return cluster > 1 ? *cl.map_shared_rank(mine, r) : *mine; };
    if (tid < G) {
        float mr[kMassMaxCluster], lr[kMassMaxCluster], M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int r = 0; r < kMassMaxCluster; ++r) {
            mr[r] = r < cluster ? theirs(&sh.ml[tid][0], r) : -INFINITY;
            lr[r] = r < cluster ? theirs(&sh.ml[tid][1], r) : 0.0f;
            M = fmaxf(M, mr[r]);
        }
#pragma unroll
        for (int r = 0; r < kMassMaxCluster; ++r)
            if (mr[r] != -INFINITY) L += lr[r] * exp2f(mr[r] - M);
        const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
        for (int r = 0; r < kMassMaxCluster; ++r) sh.weight[r][tid] = mr[r] != -INFINITY ? exp2f(mr[r] - M) * inv : 0.0f;
        sh.neg_lse[tid] = neg_log2_sum(M, L);
    }
    __syncthreads();
    T* o = (T*)p.o + ((int64_t)b * p.Hkv + h) * G * kHeadDim;
    for (int i = rank * threads + tid; i < G * kHeadDim; i += cluster * threads) {
        const int g = i / kHeadDim, d = i % kHeadDim;
        float v[kMassMaxCluster], sum = 0.0f;
#pragma unroll
        for (int r = 0; r < kMassMaxCluster; ++r) v[r] = r < cluster ? theirs(&sh.o[g][d], r) : 0.0f;
#pragma unroll
        for (int r = 0; r < kMassMaxCluster; ++r)
            if (r < cluster && sh.weight[r][g] != 0.0f) sum += v[r] * sh.weight[r][g];       // a share without tokens has no outputs
        o[i] = from_f32<T>(sum);
    }
    for (int i0 = 0; i0 < n; i0 += kEach * threads) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int i = i0 + k * threads + tid, t = i < n ? token(i) : -1;
            if (t < 0) continue;
            float sum = 0.0f;
            for (int g = 0; g < G; ++g) sum += exp2f(scores[i * G + g] + sh.neg_lse[g]);
            m.out[at + t] = t == tokens - 1 ? sum : fmaf(m.decay, before[k], sum);
        }
        if (i0 + kEach * threads < n) load(i0 + kEach * threads);
    }
    if (cluster > 1) cl.sync();               // the CTA's shared memory is read until here
}

}  // namespace ktk
