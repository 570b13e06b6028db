// Weights of a chunk's rows summed by keys, on the fifth-generation tensor cores: with the rows' denominators known,
//     sum[t] = sum over rows of 2^(s(t, row) - lse_row)
// One CTA per (sequence, kv head, 16 pages = 256 keys, part of the rows).  The scores are computed transposed,
// S^T[128 keys x 128 rows] = K . Q^T, so that a thread holds a key and sums along its own lane of tensor memory: no exchange between
// threads, and one value per key at the end.  The rows of a tile are the (token, head) pairs of 128 / G new tokens.
//
// Roles of the 320 threads:
//     warps 0..3, 4..7   exponentials and sums of the first, the second 128 keys
//     warp 8             matrix instructions: per tile of rows and 128 keys, into one of two buffers of 128 columns each
//     warp 9             the keys' pages (once), then tiles of queries (TMA) and their rows' denominators, kPmStages in flight
// Every wait is bounded.
#include "ktk_prefill_mass.cuh"
#include "ktk_umma.cuh"

#include <type_traits>

namespace ktk {

constexpr int kPmThreads = 320;
constexpr int kPmPages = 8;                               // of 128 keys
constexpr int kPmBlock = kUmRows;                         // keys of a block
constexpr int kPmTile = kUmRows * 128;                    // [128 rows][64 columns]
constexpr int kPmStages = 4;
constexpr int kPmSmem = (2 + kPmStages) * 2 * kPmTile + 1024;
constexpr int kPmTmemCols = 512;

struct PmShared {
    uint64_t k, full[kPmStages], empty[kPmStages], s[2][2], s_free[2][2];
    uint32_t tmem;
    int abort;
    alignas(16) float neg_lse[kPmStages][kUmRows];
};

// first tile of rows, counted from the first counted token, in which some row sees the token in place t
__device__ __forceinline__ int first_tile(const MassSequence& s, int tpc, int t) {
    const int tok = t - s.base_pos - s.counted;
    return tok > 0 ? tok / tpc : 0;
}

__global__ void __launch_bounds__(kPmThreads, 1)
prefill_mass_umma_kernel(const PrefillMassParams p, const __grid_constant__ CUtensorMap kv_map,
                         const __grid_constant__ CUtensorMap q_map) {
    extern __shared__ uint8_t pm_raw[];
    __shared__ __align__(16) PmShared sh;
    uint8_t* k_sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pm_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_sm = k_sm + 2 * 2 * kPmTile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    wait_for_front();
    const int h = blockIdx.x % p.Hkv, split = (int)(blockIdx.x / p.Hkv) % p.splits, group = (int)(blockIdx.x / p.Hkv) / p.splits;
    const int b = blockIdx.y, G = p.G, Hq = p.Hkv * G, tpc = kUmRows / G;
    MassSequence s;
    if (!mass_sequence(p, b, group == 0 && split == 0 && h == 0, s)) return;
    const int e0 = group * 2 * kPmPages;
    if (e0 >= s.sp.n_pages) return;                       // uniform for the CTA: nothing set up yet
    const int n_tiles = ((s.n_new - s.counted) + tpc - 1) / tpc;
    const int t_end = (split + 1) * p.tiles < n_tiles ? (split + 1) * p.tiles : n_tiles;
    if (tid == 0 && group == 0 && split == 0 && h == 0 && (n_tiles > p.splits * p.tiles || s.sp.n_pages > p.groups * 2 * kPmPages))
        report(p.status, KTK_STATUS_BAD_TABLE);           // more than the caller's bounds
    int begin[2];                                         // first tile of each block of keys
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        begin[m] = t_end;
        if (e0 + m * kPmPages < s.sp.n_pages) {
            const int f = first_tile(s, tpc, page_first_pos(e0 + m * kPmPages, s.sp.first_fill));
            begin[m] = f > split * p.tiles ? f : split * p.tiles;
            if (begin[m] > t_end) begin[m] = t_end;
        }
    }
    const int t_begin = begin[0];                         // the first block's keys are seen first
    if (t_begin >= t_end) return;

    if (warp == 8) {
        tmem_alloc(&sh.tmem, kPmTmemCols);
    } else if (warp == 9) {
        if (lane == 0) {
            prefetch_tensormap(&kv_map);
            prefetch_tensormap(&q_map);
            mbar_init(&sh.k, 1);
            for (int i = 0; i < kPmStages; ++i) {
                mbar_init(&sh.full[i], 1);
                mbar_init(&sh.empty[i], 1 + 8);           // matrix instructions, the warps that read the denominators
            }
            for (int i = 0; i < 4; ++i) {
                mbar_init(&sh.s[i >> 1][i & 1], 1);
                mbar_init(&sh.s_free[i >> 1][i & 1], 4);
            }
            sh.abort = 0;
            mbar_init_fence();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    int issued = 0;
    if (warp == 9) {
        // ---------------- copies ----------------
        const int pages = min(s.sp.n_pages - e0, 2 * kPmPages);
        const int64_t page = lane < pages ? p.kv_indices[s.sp.start + e0 + lane] : -1;
        const bool on = page >= 0 && page < p.num_pages;
        if (!on && lane < pages) report(p.status, KTK_STATUS_BAD_PAGE);
        const uint32_t n_on = __popc(__ballot_sync(0xffffffffu, on));
        if (lane == 0) {
            if (n_on) mbar_arrive_expect_tx(&sh.k, n_on * (2u * kPageSize * 128u));
            else mbar_arrive(&sh.k);
        }
        __syncwarp();
        if (on) {
            uint8_t* dst = k_sm + (lane / kPmPages) * 2 * kPmTile + (lane % kPmPages) * (kPageSize * 128);
            const int z = (int)page * (2 * kPageSize);    // token row of slot 0
            tma_load_3d(dst, &kv_map, &sh.k, 0, h, z);
            tma_load_3d(dst + kPmTile, &kv_map, &sh.k, 64, h, z);
        }
        __syncwarp();
        bool alive = true;
        for (int i = t_begin; i < t_end; ++i, ++issued) {
            const int st = issued % kPmStages, tok0 = s.counted + i * tpc;
            float nl[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = k * 32 + lane, tok = tok0 + r / G;
                nl[k] = tok < s.n_new ? -p.lse[(int64_t)(s.q0 + tok) * Hq + h * G + r % G] : 0.0f;
            }
            if (issued >= kPmStages) alive = mbar_wait_all(&sh.empty[st], ((issued / kPmStages) - 1) & 1, &sh.abort);
            if (!alive) break;
#pragma unroll
            for (int k = 0; k < 4; ++k) sh.neg_lse[st][k * 32 + lane] = nl[k];
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_expect_tx(&sh.full[st], 2 * kPmTile);
                uint8_t* dst = q_sm + st * 2 * kPmTile;
                tma_load_3d(dst, &q_map, &sh.full[st], 0, h * G, s.q0 + tok0);
                tma_load_3d(dst + kPmTile, &q_map, &sh.full[st], 64, h * G, s.q0 + tok0);
            }
            __syncwarp();
        }
    } else if (warp == 8) {
        // ---------------- matrix instructions ----------------
        const uint32_t tmem = sh.tmem, idesc = umma_idesc(kUmRows, false);
        const uint64_t k_desc = umma_desc(smem_u32(k_sm), 0, 1024), q_desc = umma_desc(smem_u32(q_sm), 0, 1024);
        bool alive = mbar_wait_all(&sh.k, 0, &sh.abort);
        for (int i = t_begin; i < t_end && alive; ++i) {
            const int n = i - t_begin, st = n % kPmStages;
            alive = mbar_wait_all(&sh.full[st], (n / kPmStages) & 1, &sh.abort);
            tc_fence_after();
            const uint64_t qb = umma_desc_at(q_desc, st * 2 * kPmTile);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (!alive || i < begin[m]) continue;
                const int j = i - begin[m];
                if (j >= 2) {
                    alive = mbar_wait_all(&sh.s_free[m][j & 1], ((j >> 1) - 1) & 1, &sh.abort);
                    tc_fence_after();
                    if (!alive) continue;
                }
                if (elect_one()) {
                    const uint64_t ka = umma_desc_at(k_desc, m * 2 * kPmTile);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            umma_f16(tmem + m * 256 + (j & 1) * 128, umma_desc_at(ka, c * kPmTile + x * 32),
                                     umma_desc_at(qb, c * kPmTile + x * 32), idesc, (c > 0 || x > 0) ? 1u : 0u);
                    umma_commit(&sh.s[m][j & 1]);
                }
                __syncwarp();
            }
            if (elect_one()) umma_commit(&sh.empty[st]);
            __syncwarp();
        }
    } else {
        // ---------------- exponentials and sums ----------------
        const int m = warp >> 2, key = tid & (kUmRows - 1);
        const int e = e0 + m * kPmPages + key / kPageSize, slot = key % kPageSize;
        const bool on = e < s.sp.n_pages && slot < (e == s.sp.n_pages - 1 ? s.sp.last_fill : (e == 0 ? s.sp.first_fill : kPageSize));
        const int t = page_first_pos(e, s.sp.first_fill) + slot;
        const int t_last = page_first_pos(e0 + (m + 1) * kPmPages, s.sp.first_fill);      // behind the block's last key
        const uint32_t my = sh.tmem + ((uint32_t)((warp & 3) * 32) << 16) + m * 256;
        const uint64_t c2 = pack2(p.scale_log2, p.scale_log2);
        float total = 0.0f, lost = 0.0f;                  // the sum, and what its rounding lost
        bool alive = true;
        for (int i = t_begin; i < t_end && alive; ++i) {
            const int n = i - t_begin, st = n % kPmStages;
            alive = mbar_wait_all(&sh.full[st], (n / kPmStages) & 1, &sh.abort);
            if (!alive) break;
            if (i >= begin[m]) {
                const int j = i - begin[m];
                alive = mbar_wait_all(&sh.s[m][j & 1], (j >> 1) & 1, &sh.abort);
                if (!alive) break;
                tc_fence_after();
                const int tok0 = s.counted + i * tpc;
                // columns that see the key, and those that are rows at all
                const int c_lo = (t - s.base_pos - tok0) * G, c_hi = (s.n_new - tok0) * G;
                const bool cut = s.base_pos + tok0 < t_last || c_hi < kUmRows;             // uniform for the block
                uint64_t acc[4] = {0, 0, 0, 0};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float v[2][32];
                    tmem_ld64(my + (j & 1) * 128 + half * 64, v[0], v[1]);
                    if (half == 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.s_free[m][j & 1]);
                    }
                    const ulonglong2* nl = reinterpret_cast<const ulonglong2*>(&sh.neg_lse[st][half * 64]);
                    auto sum = [&](auto masked) {
#pragma unroll
                        for (int c = 0; c < 64; c += 4) {
                            const ulonglong2 l = nl[c / 4];
                            float x[4];
                            unpack2(fma2(pack2(v[c / 32][c % 32], v[c / 32][c % 32 + 1]), c2, l.x), x[0], x[1]);
                            unpack2(fma2(pack2(v[c / 32][c % 32 + 2], v[c / 32][c % 32 + 3]), c2, l.y), x[2], x[3]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                x[k] = ex2(x[k]);
                                if (masked) {
                                    const int col = half * 64 + c + k;
                                    x[k] = col >= c_lo && col < c_hi ? x[k] : 0.0f;
                                }
                            }
                            acc[c / 4 % 2 * 2] = add2(acc[c / 4 % 2 * 2], pack2(x[0], x[1]));
                            acc[c / 4 % 2 * 2 + 1] = add2(acc[c / 4 % 2 * 2 + 1], pack2(x[2], x[3]));
                        }
                    };
                    if (cut) sum(std::true_type{});
                    else sum(std::false_type{});
                }
                float a, c;
                unpack2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), a, c);
                const float x = a + c - lost, y = total + x;
                lost = (y - total) - x;
                total = y;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[st]);
        }
        if (alive && on) {
            if (p.splits > 1) {
                p.partial[(((int64_t)b * p.Hkv + h) * p.splits + split) * p.groups * (2 * kPmBlock) + e * kPageSize + slot] = total;
            } else {
                const int64_t at = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
                p.m.out[at] = t >= s.base_pos ? total : fmaf(p.m.decay, p.m.in[at], total);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (sh.abort && tid == 9 * 32) {
        report(p.status, KTK_STATUS_TIMEOUT);
        volatile int never = 0;                           // copies still in flight write shared memory
        mbar_wait(&sh.k, 0, &never);
        for (int i = issued > kPmStages ? issued - kPmStages : 0; i < issued; ++i)
            mbar_wait(&sh.full[i % kPmStages], (i / kPmStages) & 1, &never);
    }
    if (warp == 8) {
        __syncwarp();
        tmem_free(sh.tmem, kPmTmemCols);
    }
}

// Adds the parts' sums, in their order
__global__ void __launch_bounds__(256)
prefill_mass_add_kernel(const PrefillMassParams p) {
    wait_for_front();
    const int b = blockIdx.z, h = blockIdx.y, tpc = kUmRows / p.G;
    MassSequence s;
    if (!mass_sequence(p, b, false, s)) return;
    const int place = blockIdx.x * 256 + threadIdx.x, e = place / kPageSize, slot = place % kPageSize;
    if (e >= s.sp.n_pages || slot >= (e == s.sp.n_pages - 1 ? s.sp.last_fill : (e == 0 ? s.sp.first_fill : kPageSize))) return;
    const int t = page_first_pos(e, s.sp.first_fill) + slot;
    const int n_tiles = ((s.n_new - s.counted) + tpc - 1) / tpc;
    const int first = first_tile(s, tpc, page_first_pos(e / (2 * kPmPages) * (2 * kPmPages), s.sp.first_fill)) / p.tiles;
    const int64_t width = (int64_t)p.groups * (2 * kPmBlock);
    const float* part = p.partial + ((int64_t)b * p.Hkv + h) * p.splits * width + place;
    float sum = 0.0f;
    for (int i = first; i < p.splits && i * p.tiles < n_tiles; ++i) sum += part[i * width];
    const int64_t at = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
    p.m.out[at] = t >= s.base_pos ? sum : fmaf(p.m.decay, p.m.in[at], sum);
}

MassPlan mass_plan(const ktk_shape* s, int max_new_tokens, int64_t max_pages, int64_t total_pages, int window) {
    MassPlan plan;
    const int tpc = kUmRows / s->group_size, counted = window > 0 && window < max_new_tokens ? window : max_new_tokens;
    const int tiles = (counted + tpc - 1) / tpc;
    plan.groups = (int)((max_pages + 2 * kPmPages - 1) / (2 * kPmPages));
    int64_t about = (int64_t)plan.groups * s->batch;      // groups of all sequences
    if (total_pages >= 0 && total_pages / (2 * kPmPages) + s->batch < about) about = total_pages / (2 * kPmPages) + s->batch;
    about *= s->num_kv_heads;
    int64_t want = (4 * (int64_t)sm_count() + about - 1) / about, most = (tiles + 3) / 4;
    if (want > most) want = most;
    if (want < 1) want = 1;
    plan.tiles = (int)((tiles + want - 1) / want);
    plan.splits = (tiles + plan.tiles - 1) / plan.tiles;
    plan.partial = plan.splits > 1 ? (size_t)s->batch * s->num_kv_heads * plan.splits * plan.groups * (2 * kPmBlock) : 0;
    return plan;
}

int launch_prefill_mass_umma(const PrefillMassParams& p, cudaStream_t st) {
    const char* who = "ktk_prefill_attention_mass";
    DecodeParams d{};                                     // only what the tensor map needs
    d.cache = p.cache; d.Hkv = p.Hkv; d.num_pages = p.num_pages;
    CUtensorMap kv_map, q_map;
    int rc = make_kv_tensor_map(&kv_map, d);
    if (rc != KTK_OK) return rc;
    const uint64_t Hq = (uint64_t)p.Hkv * p.G;
    const uint64_t dims[3] = {(uint64_t)kHeadDim, Hq, (uint64_t)p.total_new};
    const uint64_t strides[2] = {(uint64_t)kHeadDim * 2, Hq * kHeadDim * 2};
    const uint32_t box[3] = {64, (uint32_t)p.G, (uint32_t)(kUmRows / p.G)};
    rc = make_tensor_map_3d(&q_map, p.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, who);
    if (rc != KTK_OK) return rc;
    const int64_t items = (int64_t)p.groups * p.splits * p.Hkv;
    if (items > 2147483647LL) {
        set_error("%s: num_kv_heads * tokens exceed the grid limit", who);
        return KTK_ERR_TOO_LARGE;
    }
    KTK_CUDA_TRY(cudaFuncSetAttribute(prefill_mass_umma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPmSmem), who);
    KTK_CUDA_TRY(launch_behind(false, prefill_mass_umma_kernel, dim3((unsigned)items, (unsigned)p.batch), kPmThreads, kPmSmem, st, p,
                               kv_map, q_map), who);
    if (p.splits > 1)
        KTK_CUDA_TRY(launch_behind(true, prefill_mass_add_kernel, dim3((unsigned)p.groups, (unsigned)p.Hkv, (unsigned)p.batch), 256, 0,
                                   st, p), who);
    return KTK_OK;
}

}  // namespace ktk
