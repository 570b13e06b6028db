// fp32: attention of new tokens that writes its rows' denominators down, and the sums of their weights by keys (ktk_prefill_mass.cu).
// Both multiply tiles of 64 (token, head) rows with 32 keys, four by four products in a thread's registers.
#include <cooperative_groups.h>

#include <type_traits>

#include "ktk_prefill_mass.cuh"

namespace ktk {

// Where the key of the token in place t lies, in floats from the cache's start; -1: not among `tokens`, or its page is none.  A lane for each
// key of a warp's, all at once: one behind the other their page ids came at 0.6 us each.
__device__ __forceinline__ int64_t key_at(const PrefillMassParams& p, const SeqPages& sp, int h, int t, int tokens) {
    int e, slot;
    page_of_pos(t < tokens ? t : tokens - 1, sp.first_fill, e, slot);
    const int64_t page = p.kv_indices[sp.start + e];
    const bool on = page >= 0 && page < p.num_pages;
    if (!on) report(p.status, KTK_STATUS_BAD_PAGE);
    return on && t < tokens ? ((page * 2 * kPageSize + slot) * p.Hkv + h) * kHeadDim : -1;
}

// ---------------------------------------------------------------- attention
constexpr int kPaKeys = 32, kPaRows = 64;     // keys of a chunk, rows of a tile
constexpr int kPaThreads = 128;               // 16 x 8: rows tr + 16 i, keys tk + 8 j, dimensions 4 tk + 32 j
constexpr int kPaLd = kHeadDim + 4;           // floats between keys or rows in shared memory: eight of them lie in different banks
constexpr int kPaLdP = kPaKeys + 4;
constexpr int kPaSmem = ((kPaRows + 4 * kPaKeys) * kPaLd + kPaRows * kPaLdP) * 4;
constexpr int kPaMaxCluster = 8;

// One CTA, or a cluster of them that share the keys, per (sequence, kv head, 64 / G new tokens): running maximum and sum per row, two CTAs
// per SM, a chunk's keys and values on their way while the one before is multiplied.  A row's eight threads lie in one warp, so that
// its weights pass through shared memory without a barrier.
// Bound by shared memory: of a chunk's 6700 cycles of it 4100 are the scores' operands (32 bytes of them a lane for 16 FMAs), 2600 the values';
// the FMAs take 4100.  256 tokens of 32 heads over 8 behind 8192 1.06 ms (33 TFLOP/s), 2.2 by a CTA per token and kv head that
// reads all its keys; 75 and 52 of 8 over 4 behind 233 and 333 23 us, 28.
__global__ void __launch_bounds__(kPaThreads, 2)
prefill_attention_f32_kernel(const PrefillMassParams p, int cluster) {
    extern __shared__ __align__(16) float pa_smem[];
    float* rows_sm = pa_smem;                     // [row][kPaLd]; in the end the outputs
    float* kv_sm = rows_sm + kPaRows * kPaLd;     // [buffer][keys, values][key][kPaLd]
    float* p_sm = kv_sm + 4 * kPaKeys * kPaLd;    // [row][kPaLdP]; in the end maxima and sums
    wait_for_front();
    const int rank = (int)(blockIdx.x % cluster), tid = threadIdx.x, warp = tid / 32, lane = tid % 32, tk = tid % 8, tr = tid / 8;
    const int G = p.G, Hq = p.Hkv * G, shift = 31 - __clz(G), tpc = kPaRows / G;
    const int64_t item = blockIdx.x / cluster, unit = item / p.Hkv, tiles = (p.max_new + tpc - 1) / tpc;
    const int h = (int)(item % p.Hkv), b = (int)(unit % p.batch), tok0 = (int)(tiles - 1 - unit / p.batch) * tpc;       // the most keys first
    const int q0 = p.q_indptr[b], n_new = p.q_indptr[b + 1] - q0;
    if (n_new <= 0 || (tok0 >= n_new && tok0 > 0)) return;        // the same for the cluster, as all that returns here
    const SeqPages sp = seq_pages(p.kv_indptr, p.page_count, p.kv_last_page_len, p.sink_tokens, b);
    const int base_pos = sp.total - n_new;
    if (sp.bad || base_pos < 0 || q0 < 0 || q0 + (int64_t)n_new > p.total_new) {
        if (tid == 0) report(p.status, KTK_STATUS_BAD_TABLE);
        return;
    }
    const int last_tok = min(tok0 + tpc, n_new) - 1, n_keys = base_pos + last_tok + 1, n_rows = (last_tok + 1 - tok0) * G;
    const int chunks = (n_keys + kPaKeys - 1) / kPaKeys, each = (chunks + cluster - 1) / cluster;
    const int c0 = rank * each, c1 = min(c0 + each, chunks);
    const auto row_of = [&](int r) { return (int64_t)(q0 + tok0 + (r >> shift)) * Hq + h * G + (r & (G - 1)); };
    // a warp brings a row, a key or a value at a time, 16 bytes a lane; places without one get zeros
    const int64_t to_value = (int64_t)kPageSize * p.Hkv * kHeadDim;              // from a token's key to its value
    int64_t at = c0 < c1 ? key_at(p, sp, h, c0 * kPaKeys + lane, n_keys) : -1;   // of the chunk that comes next, a lane for each key
    const auto load = [&](int c) {
        float* to = kv_sm + ((c - c0) & 1) * 2 * kPaKeys * kPaLd;
#pragma unroll
        for (int i = 0; i < kPaKeys / 4; ++i) {
            const int k = warp * (kPaKeys / 4) + i;
            const int64_t from = __shfl_sync(0xffffffffu, at, k);
            const float* src = (const float*)p.cache + (from < 0 ? 0 : from + lane * 4);
            cp_async16(smem_u32(to + k * kPaLd + lane * 4), src, from < 0 ? 0 : 16);
            cp_async16(smem_u32(to + (kPaKeys + k) * kPaLd + lane * 4), from < 0 ? src : src + to_value, from < 0 ? 0 : 16);
        }
        cp_async_commit();
        if (c + 1 < c1) at = key_at(p, sp, h, (c + 1) * kPaKeys + lane, n_keys);
    };
    float m[4], l[4], o[4][16];
    int sees[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = tr + 16 * i;
        sees[i] = r < n_rows ? base_pos + tok0 + (r >> shift) : -1;
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] = 0.0f;
    }
    if (c0 < c1) {
        for (int r = warp; r < kPaRows; r += kPaThreads / 32) {
            const bool on = r < n_rows;
            cp_async16(smem_u32(rows_sm + r * kPaLd + lane * 4), (const float*)p.q + (on ? row_of(r) * kHeadDim + lane * 4 : 0), on ? 16 : 0);
        }
        load(c0);
    }
    // I: 16 rows that some row of the tile is among
    const auto multiply = [&](auto some, int c) {
        constexpr int I = decltype(some)::value;
        const int n = min(kPaKeys, n_keys - c * kPaKeys);
        const float* keys = kv_sm + ((c - c0) & 1) * 2 * kPaKeys * kPaLd;
        const float* values = keys + kPaKeys * kPaLd;
        float s[I][4] = {};                       // [row tr + 16 i][key tk + 8 j]
#pragma unroll 4
        for (int d = 0; d < kHeadDim; d += 4) {
            float4 k[4], q[I];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(keys + (tk + 8 * j) * kPaLd + d);
#pragma unroll
            for (int i = 0; i < I; ++i) q[i] = *reinterpret_cast<const float4*>(rows_sm + (tr + 16 * i) * kPaLd + d);
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(q[i].x, k[j].x, s[i][j]);
                    s[i][j] = fmaf(q[i].y, k[j].y, s[i][j]);
                    s[i][j] = fmaf(q[i].z, k[j].z, s[i][j]);
                    s[i][j] = fmaf(q[i].w, k[j].w, s[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < I; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = c * kPaKeys + tk + 8 * j <= sees[i] ? s[i][j] * p.scale_log2 : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            top = fmaxf(top, m[i]);
            const float base = top == -INFINITY ? 0.0f : top, alpha = exp2f(m[i] - base);
            m[i] = top;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = exp2f(s[i][j] - base);
                sum += w;
                p_sm[(tr + 16 * i) * kPaLdP + tk + 8 * j] = w;
            }
            l[i] = fmaf(l[i], alpha, sum);
#pragma unroll
            for (int x = 0; x < 16; ++x) o[i][x] *= alpha;
        }
        __syncwarp();
#pragma unroll 2
        for (int k0 = 0; k0 < n; k0 += 4) {
            float w[I][4];
#pragma unroll
            for (int i = 0; i < I; ++i) *reinterpret_cast<float4*>(w[i]) = *reinterpret_cast<const float4*>(p_sm + (tr + 16 * i) * kPaLdP + k0);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 v = *reinterpret_cast<const float4*>(values + (k0 + k) * kPaLd + tk * 4 + 32 * j);
#pragma unroll
                    for (int i = 0; i < I; ++i) {
                        o[i][4 * j] = fmaf(w[i][k], v.x, o[i][4 * j]);
                        o[i][4 * j + 1] = fmaf(w[i][k], v.y, o[i][4 * j + 1]);
                        o[i][4 * j + 2] = fmaf(w[i][k], v.z, o[i][4 * j + 2]);
                        o[i][4 * j + 3] = fmaf(w[i][k], v.w, o[i][4 * j + 3]);
                    }
                }
        }
    };
    for (int c = c0; c < c1; ++c) {
        cp_async_wait<0>();
        __syncthreads();
        if (c + 1 < c1) load(c + 1);
        if (n_rows <= 16) multiply(std::integral_constant<int, 1>(), c);
        else if (n_rows <= 32) multiply(std::integral_constant<int, 2>(), c);
        else multiply(std::integral_constant<int, 4>(), c);
    }
    __syncthreads();                              // queries and weights have been read
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = tr + 16 * i;
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
        if (tk == 0) reinterpret_cast<float2*>(p_sm)[r] = make_float2(m[i], l[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4*>(rows_sm + r * kPaLd + tk * 4 + 32 * j) = make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
    }
    auto cl = cooperative_groups::this_cluster();
    if (cluster > 1) cl.sync();
    else __syncthreads();
    // the CTA's part of the rows: a warp to a row, four dimensions to a lane
    const int part = kPaRows / cluster, end = min((rank + 1) * part, n_rows);
    for (int r = rank * part + warp; r < end; r += kPaThreads / 32) {
        const auto theirs = [&](const float* mine, int k) { return cluster > 1 ? cl.map_shared_rank(mine, k) : mine; };
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < cluster) ml = reinterpret_cast<const float2*>(theirs(p_sm, lane))[r];
        float4 x[kPaMaxCluster];
#pragma unroll
        for (int k = 0; k < kPaMaxCluster; ++k) x[k] = *reinterpret_cast<const float4*>(theirs(rows_sm, k < cluster ? k : 0) + r * kPaLd + lane * 4);
        float top = ml.x;
#pragma unroll
        for (int y = 1; y < kPaMaxCluster; y <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
        const float a = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - top);
        float sum = a * ml.y;
#pragma unroll
        for (int y = 1; y < kPaMaxCluster; y <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, y);
        const float L = __shfl_sync(0xffffffffu, sum, 0), M = __shfl_sync(0xffffffffu, top, 0), inv = 1.0f / L;
        float4 out = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kPaMaxCluster; ++k) {
            const float f = __shfl_sync(0xffffffffu, a, k) * inv;
            if (k >= cluster || f == 0.0f) continue;
            out.x = fmaf(x[k].x, f, out.x);
            out.y = fmaf(x[k].y, f, out.y);
            out.z = fmaf(x[k].z, f, out.z);
            out.w = fmaf(x[k].w, f, out.w);
        }
        const int64_t row = row_of(r);
        *reinterpret_cast<float4*>((float*)p.o + row * kHeadDim + lane * 4) = out;
        if (lane == 0) ((float*)p.lse)[row] = -(M + log2f(L));
    }
    if (cluster > 1) cl.sync();                   // the others read until here
}

// ---------------------------------------------------------------- sums by keys
constexpr int kPsKeys = 32, kPsRows = 64;     // keys of a CTA, rows of a tile
constexpr int kPsThreads = 128;               // 8 x 16, four keys and four rows each
constexpr int kPsLd = kHeadDim + 4;           // floats between keys or rows in shared memory: eight of them lie in different banks
constexpr int kPsSmem = (kPsKeys + 2 * kPsRows) * kPsLd * 4;

// One CTA per (sequence, kv head, 32 keys), its keys and two tiles of 64 rows in shared memory: a tile is multiplied while the next one
// comes.  Bound by shared memory: 32 cycles per dimension and tile.  Stages of 32
// dimensions instead of whole tiles were bound by the loads' latency, 2 us each.
// Where that leaves SMs idle, a cluster of CTAs takes the tiles in turn and its first one adds the sums.
__global__ void __launch_bounds__(kPsThreads)
prefill_sums_f32_kernel(const PrefillMassParams p, int chunks, int cluster) {
    extern __shared__ __align__(16) float ps_smem[];
    __shared__ float sums[kPsThreads / 8][kPsKeys], totals[kPsKeys];
    float* keys = ps_smem;                        // [key][kPsLd], then [tile][row][kPsLd]
    wait_for_front();
    const int64_t item = blockIdx.x / cluster, unit = item / chunks;
    const int part = (int)(item % chunks), rank = (int)(blockIdx.x % cluster), tid = threadIdx.x, tk = tid % 8, tr = tid / 8;
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv), G = p.G, Hq = p.Hkv * G, shift = 31 - __clz(G);    // 1, 2, 4 or 8
    MassSequence s;
    if (!mass_sequence(p, b, part == 0 && h == 0 && rank == 0, s)) return;      // the same for the cluster
    const int t0 = part * kPsKeys;
    if (t0 >= s.sp.total) return;
    // tokens that are counted and see the chunk's first key
    const int tok0 = max(s.counted, t0 - s.base_pos), n_rows = (s.n_new - tok0) * G;
    const auto row_of = [&](int r) { return (int64_t)(s.q0 + tok0 + (r >> shift)) * Hq + h * G + (r & (G - 1)); };
    // a warp brings a key or a row at a time, 16 bytes a lane; places without one get zeros
    const int warp = tid / 32, lane = tid % 32;
    const int64_t at = key_at(p, s.sp, h, t0 + lane, s.sp.total);
#pragma unroll
    for (int i = 0; i < kPsKeys / 4; ++i) {
        const int k = warp * (kPsKeys / 4) + i;
        const int64_t from = __shfl_sync(0xffffffffu, at, k);
        cp_async16(smem_u32(keys + k * kPsLd + lane * 4), (const float*)p.cache + (from < 0 ? 0 : from + lane * 4), from < 0 ? 0 : 16);
    }
    const auto load_rows = [&](int r0, int tile) {
        float* rows = keys + (kPsKeys + tile * kPsRows) * kPsLd;
        for (int r = warp; r < kPsRows; r += kPsThreads / 32) {
            const bool on = r0 + r < n_rows;
            cp_async16(smem_u32(rows + r * kPsLd + lane * 4), (const float*)p.q + (on ? row_of(r0 + r) * kHeadDim + lane * 4 : 0), on ? 16 : 0);
        }
        cp_async_commit();
    };
    load_rows(rank * kPsRows, 0);
    float sum[4] = {};
    for (int r0 = rank * kPsRows, tile = 0; r0 < n_rows; r0 += cluster * kPsRows, tile ^= 1) {
        if (r0 + cluster * kPsRows < n_rows) load_rows(r0 + cluster * kPsRows, tile ^ 1);
        else cp_async_commit();
        int sees[4];
        float lse[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + tr + 16 * i;
            sees[i] = r < n_rows ? s.base_pos + tok0 + (r >> shift) : -1;
            lse[i] = r < n_rows ? ((const float*)p.lse)[row_of(r)] : 0.0f;
        }
        cp_async_wait<1>();
        __syncthreads();
        const float* rows = keys + (kPsKeys + tile * kPsRows) * kPsLd;
        float dot[4][4] = {};                     // [row tr + 16 i][key tk + 8 j]
#pragma unroll 4
        for (int d = 0; d < kHeadDim; d += 4) {
            float4 k[4], q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(keys + (tk + 8 * j) * kPsLd + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(rows + (tr + 16 * i) * kPsLd + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    dot[i][j] = fmaf(q[i].x, k[j].x, dot[i][j]);
                    dot[i][j] = fmaf(q[i].y, k[j].y, dot[i][j]);
                    dot[i][j] = fmaf(q[i].z, k[j].z, dot[i][j]);
                    dot[i][j] = fmaf(q[i].w, k[j].w, dot[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (t0 + tk + 8 * j <= sees[i]) sum[j] += exp2f(fmaf(dot[i][j], p.scale_log2, lse[i]));
        __syncthreads();                          // the tile is free
    }
    cp_async_wait<0>();
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[tr][tk + 8 * j] = sum[j];
    __syncthreads();
    float total = 0.0f;
    if (tid < kPsKeys) {
#pragma unroll
        for (int i = 0; i < kPsThreads / 8; ++i) total += sums[i][tid];
        totals[tid] = total;
    }
    if (cluster > 1) {
        auto cl = cooperative_groups::this_cluster();
        cl.sync();
        if (rank == 0 && tid < kPsKeys)
            for (int i = 1; i < cluster; ++i) total += *cl.map_shared_rank(&totals[tid], i);
        cl.sync();                                // the others stay until theirs are read
    }
    if (rank == 0 && tid < kPsKeys && t0 + tid < s.sp.total) {
        const int t = t0 + tid;
        const int64_t to = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
        p.m.out[to] = t >= s.base_pos ? total : fmaf(p.m.decay, p.m.in[to], total);
    }
}

int launch_prefill_mass_f32(const PrefillMassParams& p, cudaStream_t st) {
    const char* who = "ktk_prefill_attention_mass";
    const int64_t tpc = kPaRows / p.G, per_seq = (p.max_new + tpc - 1) / tpc, units = (int64_t)p.batch * p.Hkv;
    const int64_t key_chunks = ((int64_t)p.max_pages * kPageSize + kPsKeys - 1) / kPsKeys, ctas = key_chunks * units;
    if (per_seq * units > 2147483647LL / kPaMaxCluster || ctas > 2147483647LL / 8) {
        set_error("%s: batch * num_kv_heads * tokens exceed the grid limit", who);
        return KTK_ERR_TOO_LARGE;
    }
    // where that leaves SMs idle, a cluster of CTAs shares a tile's keys, and the rows of a chunk of keys
    const int64_t tiles = (per_seq * p.batch < p.total_new / tpc + p.batch ? per_seq * p.batch : p.total_new / tpc + p.batch) * p.Hkv;
    int cluster = 1;
    while (cluster < kPaMaxCluster && tiles * cluster <= sm_count() && key_chunks > cluster) cluster *= 2;
    KTK_CUDA_TRY(allow_shared(prefill_attention_f32_kernel, kPaSmem), who);
    KTK_CUDA_TRY(launch_cluster(false, prefill_attention_f32_kernel, (unsigned)(per_seq * units * cluster), kPaThreads,
                                kPaSmem, cluster, st, p, cluster), who);
    const int64_t rows = (int64_t)(p.window > 0 && p.window < p.max_new ? p.window : p.max_new) * p.G;
    cluster = 1;
    while (cluster < 8 && ctas * cluster <= sm_count() && rows > (int64_t)kPsRows * cluster) cluster *= 2;
    KTK_CUDA_TRY(allow_shared(prefill_sums_f32_kernel, kPsSmem), who);
    KTK_CUDA_TRY(launch_cluster(false, prefill_sums_f32_kernel, (unsigned)(ctas * cluster), kPsThreads, kPsSmem, cluster, st, p, (int)key_chunks,
                                cluster), who);
    return KTK_OK;
}

}  // namespace ktk
