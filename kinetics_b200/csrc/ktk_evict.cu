// Eviction from a paged cache by accumulated attention weight: of every (sequence, kv head) with more than `keep` tokens the ones
// of largest mass stay, with the first and the newest.  The kept tokens behind place `keep` move into the holes in front of it.
//
// One CTA per (sequence, kv head) plans: every token has a 32-bit key whose order is that of the masses (the first and newest:
// the largest key, NaN: the smallest).  The keep-th largest key is found two bits at a time, by counting the keys that reach each of
// three thresholds, until a threshold is reached by exactly `keep` keys; tokens at exactly the last threshold stay from the lowest
// place on.  Which tokens stay is held as one bit each, and prefix sums over the bits' words number the holes and the tokens that move.
// Keys and values are copied a warp to a token, by the planning CTA or by a launch of their own (evict_move_kernel).
#include "ktk_decode.cuh"

namespace ktk {

struct EvictParams {
    void* cache;
    const int32_t* kv_indices;
    const int32_t* kv_indptr;
    const int32_t* kv_last_page_len;
    const int32_t* page_count;
    const int32_t* slot_index;
    int sink_tokens;                  // of the page table
    int Hkv;
    int64_t num_pages;
    int max_pages;
    const float* mass_in;
    float* mass_out;
    int64_t stride;
    int rows;
    const int32_t* pos_in;
    int32_t* pos_out;
    const int32_t* stored;
    const int32_t* seen;
    int keep, sink, recent;
    int32_t* count;                   // [units] tokens that move
    int32_t* from;                    // [units][max_moves] their places
    int32_t* to;                      // [units][max_moves] the holes
    int max_moves;
    int smem_keys;                    // of evict_long_kernel: keys that shared memory holds (0: none)
    int32_t* status;
};

constexpr int kEvMaxPages = 32768;

__device__ __forceinline__ uint32_t evict_key(float mass) {
    return mass != mass ? 0u : score_to_key(mass);        // NaN less than -inf (whose key is above 0)
}

// Sums over the block of three counts, up to 2^21 each, packed in 64 bits; every thread gets them.  Two buffers in turn: one barrier each.
template <int THREADS>
__device__ __forceinline__ uint64_t block_sum(uint32_t n1, uint32_t n2, uint32_t n3, uint64_t (*buf)[32], int& turn) {
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    n1 = __reduce_add_sync(0xffffffffu, n1);
    n2 = __reduce_add_sync(0xffffffffu, n2);
    n3 = __reduce_add_sync(0xffffffffu, n3);
    if (lane == 0) buf[turn][warp] = (uint64_t)n1 | (uint64_t)n2 << 21 | (uint64_t)n3 << 42;
    __syncthreads();
    const uint64_t x = lane < W ? buf[turn][lane] : 0;
    n1 = __reduce_add_sync(0xffffffffu, (uint32_t)(x & 0x1fffff));
    n2 = __reduce_add_sync(0xffffffffu, (uint32_t)(x >> 21 & 0x1fffff));
    n3 = __reduce_add_sync(0xffffffffu, (uint32_t)(x >> 42));
    turn ^= 1;
    return (uint64_t)n1 | (uint64_t)n2 << 21 | (uint64_t)n3 << 42;
}

// Exclusive prefix sum over the block's threads, and the total
template <int THREADS>
__device__ __forceinline__ uint64_t block_prefix(uint64_t x, uint64_t (*buf)[32], int& turn, uint64_t& total) {
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) buf[turn][warp] = incl;
    __syncthreads();
    uint64_t w = lane < W ? buf[turn][lane] : 0, wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, wi, o);
        if (lane >= o) wi += y;
    }
    total = __shfl_sync(0xffffffffu, wi, 31);
    const uint64_t before = __shfl_sync(0xffffffffu, wi - w, warp);
    turn ^= 1;
    return before + incl - x;
}

// A (sequence, kv head) and its tokens; false: nothing is evicted from it
struct EvictUnit {
    int n, stored, seen, start, first_fill;
    int64_t at;                                      // of its row in masses and positions
    const float* mass;
    const int32_t* pos;
    __device__ __forceinline__ int position(int t) const { return t < stored ? pos[t] : seen - n + t; }
};
__device__ __forceinline__ bool evict_unit(const EvictParams& p, int64_t unit, int most, EvictUnit& u) {
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv);
    const SeqPages sp = seq_pages(p.kv_indptr, p.page_count, p.kv_last_page_len, p.sink_tokens, b);
    const int row = p.slot_index ? p.slot_index[b] : b;
    u.n = sp.total;
    u.start = sp.start;
    u.first_fill = sp.first_fill;
    if (sp.bad || row < 0 || row >= p.rows || u.n > p.stride || sp.n_pages > p.max_pages || u.n > most) {
        if (threadIdx.x == 0) report(p.status, KTK_STATUS_BAD_TABLE);
        return false;
    }
    if (u.n <= 0) return false;
    u.at = ((int64_t)row * p.Hkv + h) * p.stride;
    u.mass = p.mass_in + u.at;
    u.pos = p.pos_in + u.at;
    u.stored = p.stored[row];
    u.seen = p.seen[row];
    return true;
}
__device__ __forceinline__ uint32_t key_at(const EvictParams& p, const EvictUnit& u, int t) {
    const int at = u.position(t);
    const float mass = u.mass[t];
    return at < p.sink || at >= u.seen - p.recent ? 0xffffffffu : evict_key(mass);
}
// What stays in its place: to be read (before anything is written), to be written
struct EvictCopy {
    float mass;
    int pos;
};
__device__ __forceinline__ EvictCopy copy_read(const EvictParams& p, const EvictUnit& u, int t) {
    return {p.mass_in == p.mass_out ? 0.0f : u.mass[t], p.pos_in == p.pos_out && t < u.stored ? 0 : u.position(t)};
}
__device__ __forceinline__ void copy_write(const EvictParams& p, const EvictUnit& u, int t, const EvictCopy& c) {
    if (p.mass_in != p.mass_out) p.mass_out[u.at + t] = c.mass;
    if (p.pos_in != p.pos_out || t >= u.stored) p.pos_out[u.at + t] = c.pos;
}

// ITEMS keys per thread, t = j * THREADS + thread: visit(j, t) for those that there are
template <int THREADS, int ITEMS, class Visit>
__device__ __forceinline__ void each_item(int n, Visit visit) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        if (j * THREADS >= n) break;                 // uniform
        visit(j, j * THREADS + (int)threadIdx.x);
    }
}

// The words of places in front of `keep`
__device__ __forceinline__ uint32_t in_front(int w, int keep) {
    return w * 32 + 32 <= keep ? 0xffffffffu : w * 32 >= keep ? 0u : (1u << (keep - w * 32)) - 1u;
}

// above, level: one bit per token, its key is above the threshold, at it.  Numbers the holes and the tokens that move, in the order of
// their places: hole(i, t), mover(i, t).  `above` becomes: the token stays.  Returns how many move.
template <int THREADS, class Hole, class Mover>
__device__ __forceinline__ int number_moves(uint32_t* above, const uint32_t* level, int words, int keep, int need, uint64_t (*buf)[32],
                                            int& turn, Hole hole, Mover mover) {
    const int tid = threadIdx.x;
    // words of a thread: consecutive ones, so that prefix sums over threads go by place
    const int each = (words + THREADS - 1) / THREADS;
    const int w0 = tid * each < words ? tid * each : words, w1 = w0 + each < words ? w0 + each : words;
    uint64_t total;
    int left = 0;                                    // how many at the threshold the thread's words may still keep
    if (need > 0) {
        uint32_t ties = 0;
        for (int w = w0; w < w1; ++w) ties += __popc(level[w]);
        left = need - (int)block_prefix<THREADS>(ties, buf, turn, total);
    }
    uint32_t holes = 0, movers = 0;
    for (int w = w0; w < w1; ++w) {
        uint32_t stay = above[w];
        if (need > 0) {
            for (uint32_t l = level[w]; l != 0 && left > 0; l &= l - 1, --left) stay |= l & (0u - l);      // the lowest places first
            above[w] = stay;
        }
        holes += __popc(~stay & in_front(w, keep));
        movers += __popc(stay & ~in_front(w, keep));
    }
    const uint64_t first = block_prefix<THREADS>((uint64_t)holes | (uint64_t)movers << 32, buf, turn, total);
    int i = (int)(uint32_t)first, k = (int)(first >> 32);
    for (int w = w0; w < w1; ++w) {
        for (uint32_t x = ~above[w] & in_front(w, keep); x != 0; x &= x - 1) hole(i++, w * 32 + __ffs((int)x) - 1);
        for (uint32_t x = above[w] & ~in_front(w, keep); x != 0; x &= x - 1) mover(k++, w * 32 + __ffs((int)x) - 1);
    }
    return (int)(uint32_t)total;
}

// Two bits of the threshold from the counts of keys that reach it plus 1, 2, 3 steps; whether exactly `keep` keys reach it now
__device__ __forceinline__ bool next_bits(uint64_t counts, int keep, int shift, uint32_t& threshold) {
    const auto count = [&](int i) { return (int)(counts >> (21 * i) & 0x1fffff); };
    const int step = count(2) >= keep ? 3 : count(1) >= keep ? 2 : count(0) >= keep ? 1 : 0;
    threshold += (uint32_t)step << shift;
    return step > 0 && count(step - 1) == keep;
}

// Tokens of a warp's copies, their loads in flight together
constexpr int kEvEach = 4;
// Copies keys and values of moves first .. first + kEvEach - 1 (of `moves`): from(i) -> to(i).  CHUNKS: 16-byte pieces of a token's key
// (as many of its value)
template <int CHUNKS, class From, class To>
__device__ __forceinline__ void copy_tokens(const EvictParams& p, int h, int start, int first_fill, int first, int moves, From from, To to) {
    constexpr int kLoads = 2 * CHUNKS / 32;
    const int lane = threadIdx.x & 31;
    uint4* cache = (uint4*)p.cache;
    // the 16-byte piece `c` of the token in place t: its key's, then its value's; -1: no such page
    const auto piece = [&](int t, int c) -> int64_t {
        int e, slot;
        page_of_pos(t, first_fill, e, slot);
        const int64_t page = __ldg(p.kv_indices + start + e);
        if (page < 0 || page >= p.num_pages) return -1;
        return (((page * 2 + c / CHUNKS) * kPageSize + slot) * p.Hkv + h) * CHUNKS + c % CHUNKS;
    };
    uint4 v[kEvEach][kLoads];
    int64_t dst[kEvEach][kLoads];
#pragma unroll
    for (int i = 0; i < kEvEach; ++i) {
        const bool on = first + i < moves;
        const int s = on ? from(first + i) : 0, d = on ? to(first + i) : 0;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            dst[i][j] = -1;
            if (!on) continue;
            const int64_t src = piece(s, j * 32 + lane);
            if (src >= 0) dst[i][j] = piece(d, j * 32 + lane);
            if (dst[i][j] >= 0) v[i][j] = cache[src];
            else report(p.status, KTK_STATUS_BAD_PAGE);
        }
    }
#pragma unroll
    for (int i = 0; i < kEvEach; ++i)
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            if (dst[i][j] >= 0) cache[dst[i][j]] = v[i][j];
}

// Sequences of at most THREADS * ITEMS tokens: keys in registers.  CHUNKS 0: keys and values are left to evict_move_kernel.
template <int THREADS, int ITEMS, int CHUNKS>
__global__ void __launch_bounds__(THREADS)
evict_kernel(const EvictParams p) {
    constexpr int kMost = THREADS * ITEMS, kWords = kMost / 32;
    __shared__ uint64_t buf[2][32];
    __shared__ uint32_t above[kWords], level[kWords];
    extern __shared__ uint16_t ev_lists[];           // [max_moves] from, [max_moves] to
    uint16_t *from = ev_lists, *to = from + p.max_moves;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    wait_for_front();
    const int64_t unit = blockIdx.x;
    EvictUnit u;
    if (!evict_unit(p, unit, kMost, u)) {
        if (CHUNKS == 0 && tid == 0) p.count[unit] = 0;
        return;
    }
    const int n = u.n, keep = p.keep;
    uint32_t key[ITEMS];
    if (n > keep) {
        each_item<THREADS, ITEMS>(n, [&](int j, int t) { key[j] = t < n ? key_at(p, u, t) : 0; });
    }
    // what stays is read early as well: the copies are written behind the search
    EvictCopy stay[ITEMS];
    const int front = n < keep ? n : keep;
    each_item<THREADS, ITEMS>(front, [&](int j, int t) { if (t < front) stay[j] = copy_read(p, u, t); });
    if (n <= keep) {
        each_item<THREADS, ITEMS>(n, [&](int j, int t) { if (t < n) copy_write(p, u, t, stay[j]); });
        if (CHUNKS == 0 && tid == 0) p.count[unit] = 0;
        return;
    }
    int turn = 0;
    uint32_t threshold = 0;                          // the largest, of the bits so far, that at least `keep` keys reach
    bool exact = false;
    for (int shift = 30; shift >= 0 && !exact; shift -= 2) {
        const uint32_t c1 = threshold + (1u << shift), c2 = threshold + (2u << shift), c3 = threshold + (3u << shift);
        uint32_t n1 = 0, n2 = 0, n3 = 0;
        each_item<THREADS, ITEMS>(n, [&](int j, int) {       // a key of 0 reaches none
            n1 += key[j] >= c1;
            n2 += key[j] >= c2;
            n3 += key[j] >= c3;
        });
        exact = next_bits(block_sum<THREADS>(n1, n2, n3, buf, turn), keep, shift, threshold);
    }
    uint32_t over = 0;
    each_item<THREADS, ITEMS>(n, [&](int j, int t) {
        const uint32_t a = __ballot_sync(0xffffffffu, t < n && (key[j] > threshold || (exact && key[j] == threshold)));
        const uint32_t l = __ballot_sync(0xffffffffu, t < n && !exact && key[j] == threshold);
        if (lane == 0) {
            above[t / 32] = a;
            level[t / 32] = l;
            over += __popc(a);
        }
    });
    const int need = keep - (int)(block_sum<THREADS>(over, 0, 0, buf, turn) & 0x1fffff);
    const int moves = number_moves<THREADS>(above, level, (n + 31) / 32, keep, need, buf, turn,
                                            [&](int i, int t) { to[i] = (uint16_t)t; }, [&](int i, int t) { from[i] = (uint16_t)t; });
    __syncthreads();
    if constexpr (CHUNKS > 0) {
        for (int i = warp * kEvEach; i < moves; i += THREADS / 32 * kEvEach)
            copy_tokens<CHUNKS>(p, (int)(unit % p.Hkv), u.start, u.first_fill, i, moves, [&](int k) { return (int)from[k]; },
                                [&](int k) { return (int)to[k]; });
    } else {
        if (tid == 0) p.count[unit] = moves;
        for (int i = tid; i < moves; i += THREADS) {
            p.from[unit * p.max_moves + i] = from[i];
            p.to[unit * p.max_moves + i] = to[i];
        }
    }
    each_item<THREADS, ITEMS>(front, [&](int j, int t) {
        if (t < front && (above[t >> 5] >> (t & 31) & 1u)) copy_write(p, u, t, stay[j]);
    });
    for (int i = tid; i < moves; i += THREADS) {
        const float mass = u.mass[from[i]];
        const int at = u.position(from[i]);
        p.mass_out[u.at + to[i]] = mass;
        p.pos_out[u.at + to[i]] = at;
    }
}

// Longer ones: keys in shared memory, or made again in every pass.
constexpr int kEvLong = 1024;
__global__ void __launch_bounds__(kEvLong)
evict_long_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t ev_smem[];
    __shared__ uint64_t buf[2][32];
    const int tid = threadIdx.x, lane = tid & 31;
    wait_for_front();
    const int64_t unit = blockIdx.x;
    EvictUnit u;
    if (!evict_unit(p, unit, kEvMaxPages * kPageSize, u)) {
        if (tid == 0) p.count[unit] = 0;
        return;
    }
    const int n = u.n, keep = p.keep;
    if (n <= keep) {
        for (int t = tid; t < n; t += kEvLong) copy_write(p, u, t, copy_read(p, u, t));
        if (tid == 0) p.count[unit] = 0;
        return;
    }
    const int words = (n + 31) / 32;
    uint32_t *above = ev_smem, *level = above + words, *keys = level + words;
    const bool held = n <= p.smem_keys;
    if (held) {
        for (int t = tid; t < n; t += kEvLong) keys[t] = key_at(p, u, t);
        __syncthreads();
    }
    const auto key_of = [&](int t) { return held ? keys[t] : key_at(p, u, t); };
    int turn = 0;
    uint32_t threshold = 0;
    bool exact = false;
    for (int shift = 30; shift >= 0 && !exact; shift -= 2) {
        const uint32_t c1 = threshold + (1u << shift), c2 = threshold + (2u << shift), c3 = threshold + (3u << shift);
        uint32_t n1 = 0, n2 = 0, n3 = 0;
        for (int t = tid; t < n; t += kEvLong) {
            const uint32_t k = key_of(t);
            n1 += k >= c1;
            n2 += k >= c2;
            n3 += k >= c3;
        }
        exact = next_bits(block_sum<kEvLong>(n1, n2, n3, buf, turn), keep, shift, threshold);
    }
    uint32_t over = 0;
    for (int t0 = tid - lane; t0 < words * 32; t0 += kEvLong) {
        const int t = t0 + lane;
        const uint32_t k = t < n ? key_of(t) : 0;
        const uint32_t a = __ballot_sync(0xffffffffu, t < n && (k > threshold || (exact && k == threshold)));
        const uint32_t l = __ballot_sync(0xffffffffu, t < n && !exact && k == threshold);
        if (lane == 0) {
            above[t0 / 32] = a;
            level[t0 / 32] = l;
            over += __popc(a);
        }
    }
    const int need = keep - (int)(block_sum<kEvLong>(over, 0, 0, buf, turn) & 0x1fffff);
    int32_t *from = p.from + unit * p.max_moves, *to = p.to + unit * p.max_moves;
    const int moves = number_moves<kEvLong>(above, level, words, keep, need, buf, turn, [&](int i, int t) { to[i] = t; },
                                            [&](int i, int t) { from[i] = t; });
    __syncthreads();
    if (tid == 0) p.count[unit] = moves;
    for (int t = tid; t < keep; t += kEvLong)
        if (above[t >> 5] >> (t & 31) & 1u) copy_write(p, u, t, copy_read(p, u, t));
    for (int i = tid; i < moves; i += kEvLong) {
        const int s = from[i], d = to[i];
        p.mass_out[u.at + d] = u.mass[s];
        p.pos_out[u.at + d] = u.position(s);
    }
}

constexpr int kEvWarps = 8;
template <int CHUNKS>
__global__ void __launch_bounds__(kEvWarps * 32)
evict_move_kernel(const EvictParams p, int parts) {
    wait_for_front();
    const int64_t unit = blockIdx.x / parts;
    const int first = ((int)(blockIdx.x % parts) * kEvWarps + (threadIdx.x >> 5)) * kEvEach;
    const int moves = p.count[unit];
    if (first >= moves) return;
    const int32_t *from = p.from + unit * p.max_moves, *to = p.to + unit * p.max_moves;
    copy_tokens<CHUNKS>(p, (int)(unit % p.Hkv), p.kv_indptr[unit / p.Hkv], p.sink_tokens > 0 ? p.sink_tokens : kPageSize, first, moves,
                        [&](int k) { return from[k]; }, [&](int k) { return to[k]; });
}

template <int THREADS, int ITEMS>
static cudaError_t launch_evict(const EvictParams& p, int64_t units, bool fused, bool f32, cudaStream_t st) {
    const auto kernel = !fused ? evict_kernel<THREADS, ITEMS, 0> : f32 ? evict_kernel<THREADS, ITEMS, 32> : evict_kernel<THREADS, ITEMS, 16>;
    const size_t smem = (size_t)p.max_moves * 2 * sizeof(uint16_t);
    if (smem > 32 * 1024) {                          // beside the static words
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    return launch_behind(units <= sm_count(), kernel, (unsigned)units, THREADS, smem, st, p);
}

static int64_t evict_max_moves(int max_pages, int keep) {
    const int64_t behind = (int64_t)max_pages * kPageSize - keep;
    return behind < 1 ? 1 : behind < keep ? behind : keep;
}

}  // namespace ktk

using namespace ktk;

extern "C" size_t ktk_evict_workspace_bytes(const ktk_shape* shape, int32_t max_pages_per_seq, int32_t keep) {
    if (check_shape(shape, "ktk_evict_workspace_bytes") != KTK_OK || shape->batch == 0 || keep < 1 || max_pages_per_seq < 1) return 0;
    const size_t units = (size_t)shape->batch * shape->num_kv_heads;
    return units * (1 + 2 * (size_t)evict_max_moves(max_pages_per_seq, keep)) * sizeof(int32_t);
}

extern "C" int ktk_evict(void* kv_cache, const int32_t* kv_indices, const int32_t* kv_indptr, const int32_t* kv_last_page_len,
                         const ktk_view* view_in, int32_t max_pages_per_seq, const ktk_mass* mass, const int32_t* positions_in,
                         int32_t* positions_out, const int32_t* stored, const int32_t* seen, int32_t keep, int32_t sink,
                         int32_t recent, void* workspace, size_t workspace_bytes, const ktk_shape* s, int32_t* status,
                         void* stream) {
    const char* who = "ktk_evict";
    int rc = check_shape(s, who);
    if (rc == KTK_OK) rc = check_view(view_in, who);
    if (rc != KTK_OK) return rc;
    if (s->batch == 0) return KTK_OK;
    if (!kv_cache || !kv_indices || !kv_indptr || !kv_last_page_len || !positions_in || !positions_out || !stored || !seen) {
        set_error("%s: null pointer argument", who);
        return KTK_ERR_ARG;
    }
    if ((rc = check_mass(mass, who)) != KTK_OK) return rc;
    const size_t bytes = (size_t)mass->rows * s->num_kv_heads * mass->stride * sizeof(float);
    if ((rc = check_apart(mass->in, mass->out, bytes, who, "mass")) != KTK_OK ||
        (rc = check_apart(positions_in, positions_out, bytes, who, "positions")) != KTK_OK ||
        (rc = check_aligned({kv_cache, workspace}, who)) != KTK_OK)
        return rc;
    if (keep < 1 || sink < 0 || recent < 0 || (int64_t)sink + recent > keep) {
        set_error("%s: keep %d, sink %d, recent %d: 1 <= keep, sink + recent <= keep", who, keep, sink, recent);
        return KTK_ERR_ARG;
    }
    if (max_pages_per_seq < 1) max_pages_per_seq = 1;
    const int64_t units = (int64_t)s->batch * s->num_kv_heads;
    if (max_pages_per_seq > kEvMaxPages || units > 2147483647LL) {
        set_error("%s: %d pages per sequence (at most %d), %lld rows", who, max_pages_per_seq, kEvMaxPages, (long long)units);
        return KTK_ERR_TOO_LARGE;
    }
    const size_t need = ktk_evict_workspace_bytes(s, max_pages_per_seq, keep);
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes needed, got %zu", who, need, workspace ? workspace_bytes : (size_t)0);
        return KTK_ERR_WORKSPACE;
    }
    const View view = make_view(view_in);
    EvictParams p;
    p.cache = kv_cache; p.kv_indices = kv_indices; p.kv_indptr = kv_indptr; p.kv_last_page_len = kv_last_page_len;
    p.page_count = view.page_count; p.slot_index = view.slot_index; p.sink_tokens = view.sink_tokens;
    p.Hkv = s->num_kv_heads; p.num_pages = s->num_pages; p.max_pages = max_pages_per_seq;
    p.mass_in = mass->in; p.mass_out = mass->out; p.stride = mass->stride; p.rows = mass->rows;
    p.pos_in = positions_in; p.pos_out = positions_out; p.stored = stored; p.seen = seen;
    p.keep = keep; p.sink = sink; p.recent = recent; p.status = status;
    p.max_moves = (int)evict_max_moves(max_pages_per_seq, keep);
    p.count = (int32_t*)workspace;
    p.from = p.count + units;
    p.to = p.from + units * p.max_moves;

    const int64_t most = (int64_t)max_pages_per_seq * kPageSize;
    cudaStream_t st = (cudaStream_t)stream;
    const int parts = (p.max_moves + kEvWarps * kEvEach - 1) / (kEvWarps * kEvEach);
    if (units * parts > 2147483647LL) {
        set_error("%s: too many tokens to move in one launch", who);
        return KTK_ERR_TOO_LARGE;
    }
    const bool fused = most <= 32768 && (units >= sm_count() || p.max_moves <= 256);
    const bool f32 = s->dtype == KTK_F32;
    if (most <= 4096) KTK_CUDA_TRY((launch_evict<512, 8>(p, units, fused, f32, st)), who);
    else if (most <= 16384) KTK_CUDA_TRY((launch_evict<1024, 16>(p, units, fused, f32, st)), who);
    else if (most <= 32768) KTK_CUDA_TRY((launch_evict<1024, 32>(p, units, fused, f32, st)), who);
    else {
        const size_t bits = (size_t)((most + 31) / 32) * 2 * sizeof(uint32_t), room = 200 * 1024;
        p.smem_keys = bits + most * sizeof(uint32_t) <= room ? (int)most : 0;
        const size_t smem = bits + (size_t)p.smem_keys * sizeof(uint32_t);
        KTK_CUDA_TRY(cudaFuncSetAttribute(evict_long_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), who);
        KTK_CUDA_TRY(launch_behind(false, evict_long_kernel, (unsigned)units, kEvLong, smem, st, p), who);
    }
    if (fused) return KTK_OK;
    const auto move = f32 ? evict_move_kernel<32> : evict_move_kernel<16>;
    KTK_CUDA_TRY(launch_behind(true, move, (unsigned)(units * parts), kEvWarps * 32, 0, st, p, parts), who);
    return KTK_OK;
}
