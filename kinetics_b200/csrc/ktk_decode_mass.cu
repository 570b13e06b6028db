// Decode attention over a paged cache that also adds up, for every cached token, the weight that it was given:
//     o[b, hq] = sum_t p_hq(t) V_t,     mass'[r, h, t] = decay mass[r, h, t] + sum over the group's heads of p_hq(t)
// with p_hq(t) = 2^(s_hq(t) - lse_hq), scores s in the log2 domain; the newest token starts from 0.
//
// A weight needs the denominator of its whole list, which is known when every key has been read.  Two forms:
//   a cluster of CTAs per (sequence, kv head) whose scores stay in shared memory: one launch (ktk_decode_mass.cuh), for lists that the
//     device holds all at once;
//   the balanced partition (bf16) or splits (fp32): the decode kernels write the scores down as they go (4 G bytes per token beside
//     the 512 of its bf16 key and value), and mass_finish_kernel turns them into weights.  It also merges the pieces of lists that
//     the decode cut.
// Bound by HBM: 48 lists of 1790 to 2303 tokens, 32 heads over 8, 80 us (5.1 TB/s), 32 of 16 K 359 (5.8 TB/s); one of 517 tokens 7.7, a
// chain of loads.
#include <type_traits>

#include "ktk_decode_mass.cuh"
#include "ktk_decode_stream.cuh"

namespace ktk {

constexpr int kMassThreads = 2 * kHeadDim;
constexpr int kMassEach = 4;                              // tokens of a thread, their loads in flight together
constexpr int kMassTokens = kMassThreads * kMassEach;     // of a CTA at a time

// The pieces of a list: `count` of them, 0 for a list that one CTA saw whole.  STREAM: behind the balanced partition; otherwise
// num_splits partials of every list.
template <bool STREAM> struct Pieces {
    int64_t first;                                        // the CTA in which the list starts; the list's number
    int count;
    __device__ __forceinline__ int64_t row(int k, int G, int g) const {
        return STREAM ? ((first + k) * 2 + (k == 0 ? 1 : 0)) * G + g : (first * G + g) * count + k;
    }
};

// One CTA per list and `rounds` times kMassTokens of its tokens, and `merges` per list for its output: one per head where there are few
// lists, each of many pieces (one sequence of 8192 tokens, 8 kv heads, 74 pieces a list: 41.5 us with one CTA for the group's heads,
// 20.6), else one (48 sequences of 2304: 80 us, 76).  A CTA's first loads, one behind the
// other, take longer than a round does: about as many CTAs as the device holds, and the next round's loads in flight.
template <typename T, bool STREAM, int G>
__global__ void __launch_bounds__(kMassThreads)
mass_finish_kernel(const StreamParams p, int chunks, int rounds, int merges, int decode_ctas) {
    __shared__ float neg_lse[G];
    const DecodeParams& d = p.d;
    const MassParams& m = p.m;
    const int tid = threadIdx.x, lane = tid & 31;
    wait_for_front();
    const int64_t unit = blockIdx.x / (chunks + merges);
    const int part = (int)(blockIdx.x % (chunks + merges));
    const int b = (int)(unit / d.Hkv), h = (int)(unit % d.Hkv);
    bool bad;
    EntryList el = entry_list(d, b, h, bad);
    const int64_t qh = ((int64_t)b * d.Hkv + h) * G;
    if (el.cnt == 0) {                                    // no token: zeros
        if (part >= chunks)
            for (int i = (part - chunks) * kMassThreads + tid; i < G * kHeadDim; i += merges * kMassThreads)
                ((T*)d.o)[qh * kHeadDim + i] = from_f32<T>(0.0f);
        return;
    }
    const int64_t start = list_position(d, m.wmax, b, h);
    if (el.cnt > m.max_pages) {                           // masses stay as they are, and the output is void
        if (tid == 0 && part == chunks) report(d.status, KTK_STATUS_BAD_TABLE);
        return;
    }
    Pieces<STREAM> pieces;
    if constexpr (STREAM) {
        int64_t total, chunk;
        stream_extent(p, decode_ctas, total, chunk);
        if (start < 0 || start + el.cnt > total) {        // starts that do not ascend: no CTA has written such pieces
            if (tid == 0 && part == chunks) report(d.status, KTK_STATUS_BAD_TABLE);
            return;
        }
        pieces.first = start / chunk;
        const int64_t last = (start + el.cnt - 1) / chunk;
        pieces.count = last == pieces.first ? 0 : (int)(last - pieces.first + 1);
    } else {
        pieces.first = unit;
        pieces.count = d.num_splits;
    }
    if (part >= chunks) {
        // a head's output: two threads to a dimension take every other piece, eight loads in flight
        if (pieces.count == 0) return;
        __shared__ float other[3][kHeadDim];
        const int dd = tid % kHeadDim, half = tid / kHeadDim;
        for (int g = part - chunks; g < G; g += merges) {
            float M = -INFINITY, L = 0.0f, O = 0.0f;
            const auto join = [&](float m2, float l2, float o2) {
                if (m2 == -INFINITY) return;              // nothing seen: its partial row is unspecified
                const float Mn = fmaxf(M, m2), a = exp2f(M - Mn), c = exp2f(m2 - Mn);
                L = L * a + l2 * c;
                O = O * a + o2 * c;
                M = Mn;
            };
            const auto some = [&](auto count, int k0) {
                constexpr int kCount = decltype(count)::value;
                float2 ml[kCount];
                float o[kCount];
#pragma unroll
                for (int i = 0; i < kCount; ++i) {
                    const int64_t at = pieces.row(min(k0 + 2 * i, pieces.count - 1), G, g);
                    ml[i] = *reinterpret_cast<const float2*>(d.ws_ml + at * 2);
                    o[i] = d.ws_o[at * kHeadDim + dd];
                }
#pragma unroll
                for (int i = 0; i < kCount; ++i)
                    if (k0 + 2 * i < pieces.count) join(ml[i].x, ml[i].y, o[i]);
            };
            some(std::integral_constant<int, 2>(), half);                       // most lists have few pieces
            for (int k0 = half + 4; k0 < pieces.count; k0 += 16) some(std::integral_constant<int, 8>(), k0);
            if (half == 1) { other[0][dd] = M; other[1][dd] = L; other[2][dd] = O; }
            __syncthreads();
            if (half == 0) {
                join(other[0][dd], other[1][dd], other[2][dd]);
                ((T*)d.o)[(qh + g) * kHeadDim + dd] = from_f32<T>(L > 0.0f ? O / L : 0.0f);
            }
            __syncthreads();
        }
        return;
    }

    const int tokens = el.cnt == 1 ? el.last : el.first + (el.cnt - 2) * kPageSize + el.last;
    const int row = m.slot_index ? m.slot_index[b] : b;
    const int t_begin = part * rounds * kMassTokens, t_end = min(t_begin + rounds * kMassTokens, tokens);
    if (t_begin >= t_end) return;
    if (row < 0 || row >= m.rows || tokens > m.stride || start < 0 || start + el.cnt > m.positions) {
        if (tid == 0 && part == 0) report(d.status, KTK_STATUS_BAD_TABLE);
        return;
    }
    const int64_t at = ((int64_t)row * d.Hkv + h) * m.stride;
    float s[kMassEach][G], before[kMassEach];
    const auto load = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kMassEach; ++i) {
            const int t = min(t0 + i * kMassThreads + tid, tokens - 1);
            // a short first page leaves places of its own block free
            const int place = t < el.first || el.cnt == 1 ? t : t + kPageSize - el.first;
            const float* from = m.scores + (start * kPageSize + place) * G;
            if constexpr (G >= 4) {
#pragma unroll
                for (int g = 0; g < G; g += 4) {
                    const float4 v = __ldcs(reinterpret_cast<const float4*>(from + g));
                    s[i][g] = v.x; s[i][g + 1] = v.y; s[i][g + 2] = v.z; s[i][g + 3] = v.w;
                }
            } else if constexpr (G == 2) {
                const float2 v = __ldcs(reinterpret_cast<const float2*>(from));
                s[i][0] = v.x; s[i][1] = v.y;
            } else {
                s[i][0] = __ldcs(from);
            }
            before[i] = m.in[at + t];
        }
    };
    load(t_begin);
    if (tid < 32) {                                       // lanes of a head: pieces lane / G, lane / G + 32 / G, ...
        const int g = lane % G;
        float M = -INFINITY, L = 0.0f;
        const auto join = [&](float m2, float l2) {
            const float Mn = fmaxf(M, m2);
            if (Mn == -INFINITY) return;
            L = L * exp2f(M - Mn) + l2 * exp2f(m2 - Mn);
            M = Mn;
        };
        for (int k = lane / G; k < pieces.count; k += 32 / G) {
            const float2 ml = *reinterpret_cast<const float2*>(d.ws_ml + pieces.row(k, G, g) * 2);
            join(ml.x, ml.y);
        }
#pragma unroll
        for (int o = G; o < 32; o <<= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, M, o), l2 = __shfl_xor_sync(0xffffffffu, L, o);
            join(m2, l2);
        }
        if (lane < G) neg_lse[lane] = pieces.count == 0 ? d.neg_lse[qh + lane] : neg_log2_sum(M, L);
    }
    __syncthreads();
    float mine[G];
#pragma unroll
    for (int g = 0; g < G; ++g) mine[g] = neg_lse[g];
    for (int t0 = t_begin; t0 < t_end; t0 += kMassTokens) {
        float sum[kMassEach], old[kMassEach];
#pragma unroll
        for (int i = 0; i < kMassEach; ++i) {
            sum[i] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) sum[i] += exp2f(s[i][g] + mine[g]);
            old[i] = before[i];
        }
        if (t0 + kMassTokens < t_end) load(t0 + kMassTokens);
#pragma unroll
        for (int i = 0; i < kMassEach; ++i) {
            const int t = t0 + i * kMassThreads + tid;
            if (t < t_end) m.out[at + t] = t == tokens - 1 ? sum[i] : fmaf(m.decay, old[i], sum[i]);
        }
    }
}

template <typename T, bool STREAM>
static int launch_finish(const StreamParams& p, int decode_ctas, cudaStream_t st) {
    const int64_t units = (int64_t)p.d.batch * p.d.Hkv, all = ((int64_t)p.m.max_pages * kPageSize + kMassTokens - 1) / kMassTokens;
    int64_t rounds = (units * all + sm_count() * 3 - 1) / (sm_count() * 3);      // CTAs that the device holds at once
    rounds = rounds < 1 ? 1 : rounds > all ? all : rounds;
    const int64_t chunks = (all + rounds - 1) / rounds, merges = units < sm_count() ? p.G : 1, ctas = (chunks + merges) * units;
    if (ctas > 2147483647LL) {
        set_error("ktk_dense_decode_mass: batch * num_kv_heads * max_pages_per_seq exceeds the grid limit");
        return KTK_ERR_TOO_LARGE;
    }
    const auto go = [&](auto kernel) {
        return launch_behind(true, kernel, (unsigned)ctas, kMassThreads, 0, st, p, (int)chunks, (int)rounds, (int)merges, decode_ctas);
    };
    KTK_CUDA_TRY(p.G == 1 ? go(mass_finish_kernel<T, STREAM, 1>) : p.G == 2 ? go(mass_finish_kernel<T, STREAM, 2>)
                 : p.G == 4 ? go(mass_finish_kernel<T, STREAM, 4>) : go(mass_finish_kernel<T, STREAM, 8>),
                 "ktk_dense_decode_mass (finish)");
    return KTK_OK;
}

int launch_mass_finish(const StreamParams& p, int decode_ctas, cudaStream_t st) { return launch_finish<__nv_bfloat16, true>(p, decode_ctas, st); }

// CTAs per list of the form that needs no workspace; 0: the other form
static int mass_cluster(const ktk_shape* s, int max_pages) {
    const int64_t units = (int64_t)s->batch * s->num_kv_heads, sms = sm_count();
    const int G = s->group_size;
    if (s->dtype == KTK_F32) {
        // as many splits as the plain decode takes, as far as a cluster goes
        const int splits = legacy_num_splits(s, max_pages);
        int c = 1;
        const auto bytes = [&](int k) { return (int64_t)(max_pages + k - 1) / k * kPageSize * G * (int64_t)sizeof(float); };
        while (c < kMassMaxCluster && (c < splits || bytes(c) > 64 * 1024)) c *= 2;
        return bytes(c) <= 160 * 1024 && splits <= 2 * kMassMaxCluster ? c : 0;
    }
    int best = 0;
    for (int c = 1; c <= kMassMaxCluster; c *= 2) {
        const int64_t per_sm = mma_mass_per_sm(4, max_pages, c, G);
        if (units * c > (per_sm < 4 ? per_sm : 4) * sms || (c > 1 && max_pages < kMmaConsumers * c)) continue;
        best = c;
    }
    if (best == 0) return 0;
    // The balanced partition where it would leave its longest CTA far fewer pages.  Pages of a CTA, even share, us with clusters and
    // balanced: 48 sequences of 2304 tokens and 8 kv heads 144, 93, 78.6 and 76.2; 55 of 1500 94, 70, 60.8 and 65.6; 48 of 2304 and one
    // kv head 18, 12, 17.5 and 27.1; one of 8192 and 8 kv heads 64, 7, 18.7 and 20.6; one of 32768 256, 28, 53.8 and 34.8.
    // It follows these, and misses the faster form in places between them.  Lists of 2049 to 2304 tokens, clusters and balanced, * what the rule
    // takes: 8 kv heads, 8 sequences 18.8* and 23.8 us, 9 30.8* and 25.0, 10 24.1 and 26.9*, 11 24.7* and 29.3, 16 29.5* and 36.2, 20 39.8 and
    // 43.0*, 24 43.0* and 46.6, 48 76.8 and 80.5*; 4 kv heads, 16 20.8* and 32.7, 20 25.9 and 35.8*, 24 27.4* and 40.2, 48 45.8* and 58.8.
    const int64_t mine = (max_pages + best - 1) / best, even = units * max_pages / (4 * sms);
    return 100 * mine <= 145 * even + 100 * (units * best >= 2 * sms ? 8 : 56) ? best : 0;
}

// Parts of the workspace, in bytes from its start
struct MassWorkspace {
    size_t lse, scores, bytes;
    int64_t positions;
    int cluster, splits;
};
static MassWorkspace mass_workspace(const ktk_shape* s, int max_pages, int64_t total_pages) {
    MassWorkspace w{};
    w.cluster = mass_cluster(s, max_pages);
    if (w.cluster > 0) {
        w.splits = w.cluster;
        return w;
    }
    const int64_t padded = (int64_t)s->batch * max_pages;
    if (total_pages < 0 || total_pages > padded) total_pages = padded;
    const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    w.splits = policy_num_splits(s, KTK_VARIANT_AUTO, max_pages);
    const size_t rows = (size_t)s->batch * s->num_kv_heads * s->group_size;
    w.positions = total_pages * s->num_kv_heads;
    w.lse = up(w.splits == KTK_SPLITS_BALANCED ? ktk_decode_workspace_bytes(s, w.splits)
                                               : rows * w.splits * (2 + kHeadDim) * sizeof(float));
    w.scores = w.lse + up(rows * sizeof(float));
    w.bytes = w.scores + up((size_t)w.positions * kPageSize * s->group_size * sizeof(float));
    return w;
}

}  // namespace ktk

using namespace ktk;

extern "C" size_t ktk_decode_mass_workspace_bytes(const ktk_shape* shape, int32_t max_pages_per_seq, int64_t total_pages) {
    if (check_shape(shape, "ktk_decode_mass_workspace_bytes") != KTK_OK || shape->batch == 0) return 0;
    return mass_workspace(shape, max_pages_per_seq < 1 ? 1 : max_pages_per_seq, total_pages).bytes;
}

extern "C" int ktk_dense_decode_mass(const void* q, const void* kv_cache, const int32_t* kv_indices,
                                     const int32_t* kv_indptr, const int32_t* kv_last_page_len, const ktk_view* view_in,
                                     int32_t max_pages_per_seq, int64_t total_pages, float sm_scale, const ktk_mass* mass,
                                     void* o, void* workspace, size_t workspace_bytes, const ktk_shape* s, int32_t* status,
                                     void* stream) {
    const char* who = "ktk_dense_decode_mass";
    int rc = check_shape(s, who);
    if (rc == KTK_OK) rc = check_view(view_in, who);
    if (rc != KTK_OK) return rc;
    if (s->batch == 0) return KTK_OK;
    if (!q || !kv_cache || !kv_indices || !kv_indptr || !kv_last_page_len || !o) {
        set_error("%s: null pointer argument", who);
        return KTK_ERR_ARG;
    }
    if ((rc = check_mass(mass, who)) != KTK_OK || (rc = check_aligned({q, kv_cache, o, workspace}, who)) != KTK_OK ||
        (rc = check_apart(mass->in, mass->out, (size_t)mass->rows * s->num_kv_heads * mass->stride * sizeof(float), who, "mass")) != KTK_OK)
        return rc;
    if (max_pages_per_seq < 1) max_pages_per_seq = 1;
    if (max_pages_per_seq > kMassMaxPages) {
        set_error("%s: %d pages per sequence, at most %d", who, max_pages_per_seq, kMassMaxPages);
        return KTK_ERR_TOO_LARGE;
    }
    const View view = make_view(view_in);
    if (view.page_count) total_pages = -1;                // padded
    const MassWorkspace w = mass_workspace(s, max_pages_per_seq, total_pages);
    if (w.bytes > 0 && (workspace == nullptr || workspace_bytes < w.bytes)) {
        set_error("%s: workspace of %zu bytes needed, got %zu", who, w.bytes, workspace ? workspace_bytes : (size_t)0);
        return KTK_ERR_WORKSPACE;
    }
    if ((int64_t)s->batch * s->num_kv_heads * (w.splits > 0 ? w.splits : 1) > 2147483647LL) {
        set_error("%s: batch * num_kv_heads * splits exceeds the grid limit", who);
        return KTK_ERR_TOO_LARGE;
    }
    DecodeParams p{};
    p.q = q; p.cache = kv_cache; p.o = o; p.entries = kv_indices;
    p.kv_indptr = kv_indptr; p.kv_last_page_len = kv_last_page_len;
    p.sink_tokens = view.sink_tokens; p.local_tokens = view.local_tokens; p.page_count = view.page_count;
    p.topk = -1; p.batch = s->batch; p.Hkv = s->num_kv_heads; p.num_pages = s->num_pages;
    p.scale_log2 = sm_scale * kLog2e;
    p.num_splits = w.splits;
    MassParams m{};
    m.in = mass->in; m.out = mass->out; m.stride = mass->stride; m.rows = mass->rows; m.slot_index = view.slot_index;
    m.decay = mass->decay; m.wmax = max_pages_per_seq; m.max_pages = max_pages_per_seq;
    p.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    if (w.cluster > 0)
        return s->dtype == KTK_F32 ? launch_decode_simt_mass(p, m, s->group_size, true, st) : launch_decode_mma_mass(p, m, s->group_size, st);
    const bool balanced = w.splits == KTK_SPLITS_BALANCED;
    const int64_t rows = balanced ? (int64_t)(ktk_decode_workspace_bytes(s, w.splits) / ((2 + kHeadDim) * sizeof(float)))
                                  : (int64_t)s->batch * s->num_kv_heads * s->group_size * w.splits;
    char* ws = (char*)workspace;
    p.ws_ml = (float*)ws;
    p.ws_o = (float*)ws + rows * 2;
    p.neg_lse = (float*)(ws + w.lse);
    m.scores = (float*)(ws + w.scores);
    m.positions = w.positions;
    if (balanced) return launch_decode_stream_mass(p, m, s->group_size, max_pages_per_seq, st);
    rc = launch_decode_simt_mass(p, m, s->group_size, false, st);
    if (rc != KTK_OK) return rc;
    StreamParams sp{};
    sp.d = p;
    sp.m = m;
    sp.G = s->group_size;
    return launch_finish<float, false>(sp, 0, st);
}
