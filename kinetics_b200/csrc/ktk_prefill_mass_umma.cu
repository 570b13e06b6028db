// Weights of a chunk's rows summed by keys, on the fifth-generation tensor cores: with the rows' denominators known,
//     sum[t] = sum over rows of 2^(s(t, row) - lse_row)
// One CTA per (sequence, kv head, 16 pages = 256 keys, part of the rows that see them), two CTAs per SM.  The scores are computed
// transposed, S^T[128 keys x 64 rows] = K . Q^T, so that a thread holds a key and sums along its own lane of tensor memory: no exchange
// between threads, and one value per key at the end.  The rows of a tile are the (token, head) pairs of 64 / G new tokens.
// A row's denominator is the same for all threads; read from shared memory it would take as much of it as the matrix instructions do
// (a word for each of 32 lanes: 4 cycles per four columns and warp).  So it is one more step of the product: minus lse over the
// scale, as three bf16 that add up to its 24 bits (written so by the attention kernel), times keys of three ones.
//
// The keys go on to tensor memory, an instruction's other operand then is all that it reads from shared memory: 32 cycles for 64 rows,
// 48 with the keys there.
//
// Roles of the 320 threads:
//     warps 0..3, 4..7   the first, the second 128 keys to tensor memory; exponentials and sums
//     warp 8             matrix instructions: per tile of rows and 128 keys, as soon as the last tile's scores are in registers
//     warp 9             TMA: the keys' pages (once), then tiles of queries and their rows' denominators, kPmStages in flight, all but the
//                        first kPmFirst of them where the keys were
// Every wait is bounded.
//
// Per 128 keys and 128 rows: 1024 cycles of the special-function units (16 exponentials a cycle) without kPmPoly, some 600 of the tensor
// cores.  A prompt of 8192 tokens, 32 heads over 8: 279 us, special-function pipe 74 %, tensor pipe 55 %; 306 with the keys in
// shared memory and no polynomials, 354 with denominators read from there too, 466 with one CTA per SM and unequal parts.
#include "ktk_prefill_mass.cuh"
#include "ktk_umma.cuh"

#include <type_traits>

namespace ktk {

constexpr int kPmThreads = 320;
constexpr int kPmPages = 8;                               // of 128 keys
constexpr int kPmBlock = kUmRows;                         // keys of a block
constexpr int kPmRows = 64;                               // rows of a tile
constexpr int kPmKTile = kPmBlock * 128, kPmQTile = kPmRows * 128;      // [128 keys], [64 rows][64 columns]
constexpr int kPmOnes = kPmBlock * 16, kPmLse = kPmRows * 16;         // [128 keys], [64 rows][8 columns]: the first 8 of the last step
constexpr int kPmStage = 2 * kPmQTile + kPmLse;
constexpr int kPmFirst = 2, kPmStages = 5;
static_assert((kPmStages - kPmFirst) * kPmStage <= 4 * kPmKTile, "stages where the keys were");
constexpr int kPmSmem = 4 * kPmKTile + kPmFirst * kPmStage + 2 * kPmOnes + 1024;
constexpr int kPmTmemCols = 256, kPmColS = 128;          // keys m at column 64 m, scores m at 128 + 64 m
constexpr int kPmPoly = 2;                                // of eight pairs of exponentials; 0, 1, 2, 3, 4: 300, 281, 277, 290, 317 us

struct PmShared {
    uint64_t k, k_moved, full[kPmStages], empty[kPmStages], s[2], s_free[2];
    uint32_t tmem;
    int abort;
};

// Operand descriptor without a swizzle, K-major: rows of 16 bytes, eight to 128 bytes; `next`: bytes to the next 8 columns
__device__ __forceinline__ uint64_t umma_desc_rows16(uint32_t saddr, uint32_t next) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)((next >> 4) & 0x3FFFu) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

// first tile of rows, counted from the first counted token, in which some row sees the token in place t
__device__ __forceinline__ int first_tile(const MassSequence& s, int tpc, int t) {
    const int tok = t - s.base_pos - s.counted;
    return tok > 0 ? tok / tpc : 0;
}

// 2^x for x <= 126 (smaller than 2^-126: that), two at a time: x = n + f, 2^f by the polynomial of degree 5 with the least relative error
// over [-1/2, 1/2] (7.5e-8; 2.3e-7 in fp32), times 2^n.  n + 1.5 2^23 has n in its lowest bits.  NaN stays NaN.
__device__ __forceinline__ float at_least(float x, float low) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(low));
    return r;
}
__device__ __forceinline__ void exp2_poly(float& x, float& y) {
    const float magic = 12582912.0f;
    const uint64_t v = pack2(at_least(x, -126.0f), at_least(y, -126.0f));
    const uint64_t t = add2(v, pack2(magic, magic)), n = add2(t, pack2(-magic, -magic)), f = fma2(n, pack2(-1.0f, -1.0f), v);
    uint64_t r = fma2(f, pack2(0.0013276472f, 0.0013276472f), pack2(0.009675541f, 0.009675541f));
    r = fma2(r, f, pack2(0.05550713f, 0.05550713f));
    r = fma2(r, f, pack2(0.2402212f, 0.2402212f));
    r = fma2(r, f, pack2(0.69314694f, 0.69314694f));
    r = fma2(r, f, pack2(1.0000001f, 1.0000001f));
    float t0, t1;
    unpack2(t, t0, t1);
    const auto power = [](float n) { return __uint_as_float((__float_as_uint(n) << 23) + 0x3f800000u); };
    unpack2(mul2(r, pack2(power(t0), power(t1))), x, y);
}

// The group-th 16 pages among those of all sequences with new tokens: its sequence and its number there, by a whole warp; false: there
// are fewer.
__device__ __forceinline__ bool find_group(const PrefillMassParams& p, int group, int& b, int& g) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int i = b0 + lane;
        int mine = 0;
        if (i < p.batch && p.q_indptr[i + 1] > p.q_indptr[i]) {
            const int pages = p.page_count ? p.page_count[i] : p.kv_indptr[i + 1] - p.kv_indptr[i];
            mine = pages > p.max_pages ? 1 : pages > 0 ? (pages + 2 * kPmPages - 1) / (2 * kPmPages) : 0;     // too many: one to say so
        }
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const unsigned here = __ballot_sync(0xffffffffu, group < upto);
        if (here != 0) {
            const int at = __ffs((int)here) - 1;
            b = b0 + at;
            g = group - __shfl_sync(0xffffffffu, upto - mine, at);
            return true;
        }
        group -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// Whether all groups of the sequence of group `item` are among the launch's: else its masses stay as they are
__device__ __forceinline__ bool all_groups(const MassSequence& s, int item, int group, int items) {
    return item - group + (s.sp.n_pages + 2 * kPmPages - 1) / (2 * kPmPages) <= items;
}

// Tiles of rows of a group of pages: those from the first that sees its first key on, cut into equal parts
struct PmTiles {
    int first, all, each;
};
__device__ __forceinline__ PmTiles tiles_of(const PrefillMassParams& p, const MassSequence& s, int g, int tpc) {
    PmTiles t;
    t.all = ((s.n_new - s.counted) + tpc - 1) / tpc;
    t.first = first_tile(s, tpc, page_first_pos(g * 2 * kPmPages, s.sp.first_fill));
    t.each = (t.all - t.first + p.splits - 1) / p.splits;
    return t;
}

__global__ void __launch_bounds__(kPmThreads, 2)
prefill_mass_umma_kernel(const PrefillMassParams p, const __grid_constant__ CUtensorMap kv_map,
                         const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap lse_map) {
    extern __shared__ uint8_t pm_raw[];
    __shared__ __align__(16) PmShared sh;
    uint8_t* k_sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pm_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* first_sm = k_sm + 4 * kPmKTile;
    uint8_t* ones_sm = first_sm + kPmFirst * kPmStage;    // then as many zeros: the other 8 columns of the last step
    const auto stage = [&](int st) { return st < kPmFirst ? first_sm + st * kPmStage : k_sm + (st - kPmFirst) * kPmStage; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    wait_for_front();
    const int h = blockIdx.x % p.Hkv, split = (int)(blockIdx.x / p.Hkv) % p.splits, item = (int)(blockIdx.x / p.Hkv) / p.splits;
    const int G = p.G, Hq = p.Hkv * G, tpc = kPmRows / G;
    int b, group;
    const int items = (int)(gridDim.x / p.Hkv) / p.splits;
    if (item == items - 1 && h == 0 && split == 0 && find_group(p, items, b, group) && tid == 0)
        report(p.status, KTK_STATUS_BAD_TABLE);           // more than the caller's bounds
    if (!find_group(p, item, b, group)) return;           // uniform for the CTA, as all that follows: nothing set up yet
    MassSequence s;
    if (!mass_sequence(p, b, group == 0 && split == 0 && h == 0, s) || !all_groups(s, item, group, items)) return;
    const int e0 = group * 2 * kPmPages;
    const PmTiles tiles = tiles_of(p, s, group, tpc);
    const int t_begin = tiles.first + split * tiles.each, t_end = min(t_begin + tiles.each, tiles.all);
    if (t_begin >= t_end) return;
    int begin[2] = {t_begin, t_end};                      // first tile of each block of keys: the first block's are seen first
    if (e0 + kPmPages < s.sp.n_pages)
        begin[1] = min(max(first_tile(s, tpc, page_first_pos(e0 + kPmPages, s.sp.first_fill)), t_begin), t_end);

    if (warp == 8) {
        tmem_alloc(&sh.tmem, kPmTmemCols);
    } else if (warp == 9) {
        if (lane == 0) {
            prefetch_tensormap(&kv_map);
            prefetch_tensormap(&q_map);
            prefetch_tensormap(&lse_map);
            mbar_init(&sh.k, 1);
            for (int i = 0; i < kPmStages; ++i) {
                mbar_init(&sh.full[i], 1);
                mbar_init(&sh.empty[i], 1);
            }
            mbar_init(&sh.k_moved, 8);
            for (int m = 0; m < 2; ++m) {
                mbar_init(&sh.s[m], 1);
                mbar_init(&sh.s_free[m], 4);
            }
            sh.abort = 0;
            mbar_init_fence();
        }
    } else if (tid < kPmBlock) {
        const uint4 ones = make_uint4(0x3F803F80u, 0x00003F80u, 0u, 0u);
        *reinterpret_cast<uint4*>(ones_sm + tid * 16) = ones;
        *reinterpret_cast<uint4*>(ones_sm + kPmOnes + tid * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async();
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
            uint8_t* dst = k_sm + (lane / kPmPages) * 2 * kPmKTile + (lane % kPmPages) * (kPageSize * 128);
            const int z = (int)page * (2 * kPageSize);    // token row of slot 0
            tma_load_3d(dst, &kv_map, &sh.k, 0, h, z);
            tma_load_3d(dst + kPmKTile, &kv_map, &sh.k, 64, h, z);
        }
        __syncwarp();
        if (lane == 0) {
            bool alive = true;
            for (int i = t_begin; i < t_end; ++i, ++issued) {
                const int st = issued % kPmStages, token = s.q0 + s.counted + i * tpc;
                if (issued == kPmFirst) alive = mbar_wait_fast(&sh.k_moved, 0, &sh.abort);
                if (issued >= kPmStages) alive = alive && mbar_wait_fast(&sh.empty[st], ((issued / kPmStages) - 1) & 1, &sh.abort);
                if (!alive) break;
                uint8_t* dst = stage(st);
                mbar_arrive_expect_tx(&sh.full[st], kPmStage);
                tma_load_3d(dst, &q_map, &sh.full[st], 0, h * G, token);
                tma_load_3d(dst + kPmQTile, &q_map, &sh.full[st], 64, h * G, token);
                tma_load_3d(dst + 2 * kPmQTile, &lse_map, &sh.full[st], 0, h * G, token);
            }
        }
        __syncwarp();
    } else if (warp == 8) {
        // ---------------- matrix instructions ----------------
        const uint32_t tmem = sh.tmem, idesc = umma_idesc(kPmRows, false);
        const uint64_t q_desc = umma_desc(smem_u32(k_sm), 0, 1024), ones_desc = umma_desc_rows16(smem_u32(ones_sm), kPmOnes);
        bool alive = mbar_wait_all(&sh.k_moved, 0, &sh.abort);
        for (int i = t_begin; i < t_end && alive; ++i) {
            const int n = i - t_begin, st = n % kPmStages;
            alive = mbar_wait_all(&sh.full[st], (n / kPmStages) & 1, &sh.abort);
            tc_fence_after();
            const uint64_t qb = umma_desc_at(q_desc, (uint32_t)(stage(st) - k_sm));
            const uint32_t lse_at = smem_u32(stage(st) + 2 * kPmQTile);
            const uint64_t lse_desc = umma_desc_rows16(lse_at, smem_u32(ones_sm + kPmOnes) - lse_at);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (!alive || i < begin[m]) continue;
                const int j = i - begin[m];
                if (j > 0) {
                    alive = mbar_wait_all(&sh.s_free[m], (j - 1) & 1, &sh.abort);
                    tc_fence_after();
                    if (!alive) continue;
                }
                if (elect_one()) {
                    const uint32_t to = tmem + kPmColS + m * kPmRows;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            umma_f16_ts(to, tmem + m * 64 + c * 32 + x * 8, umma_desc_at(qb, c * kPmQTile + x * 32), idesc,
                                        (c > 0 || x > 0) ? 1u : 0u);
                    // last: what was added before is rounded to the size of a score, not of lse
                    umma_f16(to, ones_desc, lse_desc, idesc, 1u);
                    umma_commit(&sh.s[m]);
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
        const uint32_t my = sh.tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint64_t c2 = pack2(p.scale_log2, p.scale_log2);
        float total = 0.0f, lost = 0.0f;                  // the sum, and what its rounding lost
        bool alive = mbar_wait_all(&sh.k, 0, &sh.abort);
        if (alive) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {                 // a row of 64 columns, two to a word
                uint32_t w[32];
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    *reinterpret_cast<uint4*>(w + 4 * x) = *reinterpret_cast<const uint4*>(k_sm + (2 * m + c) * kPmKTile + swz(key, x));
                tmem_st32_u32(my + m * 64 + c * 32, w);
            }
            tmem_st_wait();
            tc_fence_before();
            fence_proxy_async();                          // TMA writes there next
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_moved);
        }
        for (int i = begin[m]; i < t_end && alive; ++i) {
            const int j = i - begin[m], tok0 = s.counted + i * tpc;
            alive = mbar_wait_all(&sh.s[m], j & 1, &sh.abort);
            if (!alive) break;
            tc_fence_after();
            float v[2][32];
            tmem_ld64(my + kPmColS + m * kPmRows, v[0], v[1]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.s_free[m]);
            // columns that see the key, and those that are rows at all
            const int c_lo = max(t - s.base_pos - tok0, 0) * G, c_hi = (s.n_new - tok0) * G;
            uint64_t acc[4] = {0, 0, 0, 0};
            auto sum = [&](auto masked) {
#pragma unroll
                for (int col = 0; col < kPmRows; col += 2) {
                    const int pair = col / 2 % 8;
                    float x, y;
                    unpack2(mul2(pack2(v[col / 32][col % 32], v[col / 32][col % 32 + 1]), c2), x, y);
                    if (pair * kPmPoly % 8 + kPmPoly > 7) {              // kPmPoly of eight, evenly spread
                        exp2_poly(x, y);
                    } else {
                        x = ex2(x);
                        y = ex2(y);
                    }
                    if (masked) {
                        x = col >= c_lo && col < c_hi ? x : 0.0f;
                        y = col + 1 >= c_lo && col + 1 < c_hi ? y : 0.0f;
                    }
                    acc[col / 2 % 4] = add2(acc[col / 2 % 4], pack2(x, y));
                }
            };
            if (s.base_pos + tok0 < t_last || c_hi < kPmRows) sum(std::true_type{});      // uniform for the block
            else sum(std::false_type{});
            float a, c;
            unpack2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), a, c);
            const float x = a + c - lost, y = total + x;
            lost = (y - total) - x;
            total = y;
        }
        if (alive && on) {
            if (p.splits > 1) {
                p.partial[(((int64_t)item * p.Hkv + h) * p.splits + split) * (2 * kPmBlock) + m * kPmBlock + key] = total;
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

// Adds the parts' sums, in their order: a CTA per group of pages and kv head
__global__ void __launch_bounds__(2 * kPmBlock)
prefill_mass_add_kernel(const PrefillMassParams p) {
    wait_for_front();
    const int h = blockIdx.x % p.Hkv, item = blockIdx.x / p.Hkv, tid = threadIdx.x;
    int b, group;
    MassSequence s;
    if (!find_group(p, item, b, group) || !mass_sequence(p, b, false, s) || !all_groups(s, item, group, (int)(gridDim.x / p.Hkv))) return;
    const int e = group * 2 * kPmPages + tid / kPageSize, slot = tid % kPageSize;
    if (e >= s.sp.n_pages || slot >= (e == s.sp.n_pages - 1 ? s.sp.last_fill : (e == 0 ? s.sp.first_fill : kPageSize))) return;
    const int t = page_first_pos(e, s.sp.first_fill) + slot;
    const PmTiles tiles = tiles_of(p, s, group, kPmRows / p.G);
    const float* part = p.partial + ((int64_t)item * p.Hkv + h) * p.splits * (2 * kPmBlock) + tid;
    float sum = 0.0f;
#pragma unroll 4
    for (int i = 0; i < p.splits; ++i)
        if (tiles.first + i * tiles.each < tiles.all) sum += part[i * (2 * kPmBlock)];
    const int64_t at = ((int64_t)s.row * p.Hkv + h) * p.m.stride + t;
    p.m.out[at] = t >= s.base_pos ? sum : fmaf(p.m.decay, p.m.in[at], sum);
}

// Parts: some four rounds of the CTAs that the device holds (two per SM), of 512 rows at least.  The parts of early keys, which the most
// rows see, start first.
MassPlan mass_plan(const ktk_shape* s, int max_new_tokens, int64_t max_pages, int64_t total_pages, int window) {
    MassPlan plan;
    const int64_t each = (max_pages + 2 * kPmPages - 1) / (2 * kPmPages);
    plan.groups = each * s->batch;
    if (total_pages >= 0 && total_pages / (2 * kPmPages) + s->batch < plan.groups) plan.groups = total_pages / (2 * kPmPages) + s->batch;
    const int64_t rows = (int64_t)(window > 0 && window < max_new_tokens ? window : max_new_tokens) * s->group_size;
    const int64_t ctas = plan.groups * s->num_kv_heads;
    int64_t splits = (8 * (int64_t)sm_count() + ctas - 1) / ctas, most = (rows + 511) / 512;
    if (splits > most) splits = most;
    plan.splits = splits < 1 ? 1 : (int)splits;
    plan.partial = plan.splits > 1 ? (size_t)ctas * plan.splits * (2 * kPmBlock) : 0;
    return plan;
}

int launch_prefill_mass_umma(const PrefillMassParams& p, int64_t groups, cudaStream_t st) {
    const char* who = "ktk_prefill_attention_mass";
    DecodeParams d{};                                     // only what the tensor map needs
    d.cache = p.cache; d.Hkv = p.Hkv; d.num_pages = p.num_pages;
    CUtensorMap kv_map, q_map, lse_map;
    int rc = make_kv_tensor_map(&kv_map, d);
    if (rc != KTK_OK) return rc;
    const uint64_t Hq = (uint64_t)p.Hkv * p.G;
    const uint64_t dims[3] = {(uint64_t)kHeadDim, Hq, (uint64_t)p.total_new};
    const uint64_t strides[2] = {(uint64_t)kHeadDim * 2, Hq * kHeadDim * 2};
    const uint32_t box[3] = {64, (uint32_t)p.G, (uint32_t)(kPmRows / p.G)};
    rc = make_tensor_map_3d(&q_map, p.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, who);
    if (rc != KTK_OK) return rc;
    const uint64_t lse_dims[3] = {8, Hq, (uint64_t)p.total_new}, lse_strides[2] = {16, Hq * 16};
    const uint32_t lse_box[3] = {8, (uint32_t)p.G, (uint32_t)(kPmRows / p.G)};
    rc = make_tensor_map_3d(&lse_map, p.lse, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, lse_dims, lse_strides, lse_box, CU_TENSOR_MAP_SWIZZLE_NONE,
                            who);
    if (rc != KTK_OK) return rc;
    const int64_t units = groups * p.Hkv;
    if (units * p.splits > 2147483647LL) {
        set_error("%s: num_kv_heads * tokens exceed the grid limit", who);
        return KTK_ERR_TOO_LARGE;
    }
    KTK_CUDA_TRY(allow_shared(prefill_mass_umma_kernel, kPmSmem), who);
    KTK_CUDA_TRY(launch_behind(true, prefill_mass_umma_kernel, (unsigned)(units * p.splits), kPmThreads, kPmSmem, st, p, kv_map, q_map,
                               lse_map), who);
    if (p.splits > 1)
        KTK_CUDA_TRY(launch_behind(true, prefill_mass_add_kernel, (unsigned)units, 2 * kPmBlock, 0, st, p), who);
    return KTK_OK;
}

}  // namespace ktk
