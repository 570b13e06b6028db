// Eviction from a paged cache by accumulated attention weight: of every (sequence, kv head) with more than `keep` tokens the ones
// of largest mass stay, with the first and the newest.  The kept tokens behind place `keep` move into the holes in front of it.
//
// evict_plan_kernel, one CTA per (sequence, kv head): every token has a 32-bit key whose order is that of the masses (the
// first and newest: the largest key, NaN: the smallest).  The keep-th largest key is found two bits at a time, by counting the keys
// that reach each of three thresholds; tokens at exactly that key stay from the lowest place on.  Which tokens stay is held as one bit
// each, and prefix sums over the bits' words number the holes and the tokens that move.
// evict_move_kernel copies keys and values, a warp to a token.
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
    int smem_keys;                    // keys that shared memory holds (0: they are made again in every pass)
    int32_t* status;
};

constexpr int kEvMaxPages = 32768;

__device__ __forceinline__ uint32_t evict_key(float mass) {
    return mass != mass ? 0u : score_to_key(mass);        // NaN less than -inf (whose key is above 0)
}

// Sum over the block of up to three 21-bit counts packed in 64 bits; every thread gets it.  Two buffers in turn: one barrier each.
template <int THREADS>
__device__ __forceinline__ uint64_t block_sum(uint64_t x, uint64_t (*buf)[32], int& turn) {
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) buf[turn][warp] = x;
    __syncthreads();
    x = lane < W ? buf[turn][lane] : 0;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    x = __shfl_sync(0xffffffffu, x, 0);
    turn ^= 1;
    return x;
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

template <int THREADS>
__global__ void __launch_bounds__(THREADS)
evict_plan_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t ev_smem[];
    __shared__ uint64_t buf[2][32];
    const int tid = threadIdx.x, lane = tid & 31;
    wait_for_front();
    const int64_t unit = blockIdx.x;
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv);
    const SeqPages sp = seq_pages(p.kv_indptr, p.page_count, p.kv_last_page_len, p.sink_tokens, b);
    const int n = sp.total, row = p.slot_index ? p.slot_index[b] : b;
    const bool bad = sp.bad || row < 0 || row >= p.rows || n > p.stride || sp.n_pages > p.max_pages;
    if (bad || n <= 0) {
        if (tid == 0) {
            if (bad) report(p.status, KTK_STATUS_BAD_TABLE);
            p.count[unit] = 0;
        }
        return;
    }
    const int64_t at = ((int64_t)row * p.Hkv + h) * p.stride;
    const float* mass = p.mass_in + at;
    const int32_t* pos = p.pos_in + at;
    const int stored = p.stored[row], seen = p.seen[row], keep = p.keep;
    const auto position = [&](int t) { return t < stored ? pos[t] : seen - n + t; };
    const bool same_mass = p.mass_in == p.mass_out, same_pos = p.pos_in == p.pos_out;
    // what stays in its place
    const auto copy = [&](int t) {
        if (!same_mass) p.mass_out[at + t] = mass[t];
        if (!same_pos || t >= stored) p.pos_out[at + t] = position(t);
    };
    if (n <= keep) {
        for (int t = tid; t < n; t += THREADS) copy(t);
        if (tid == 0) p.count[unit] = 0;
        return;
    }
    const int words = (n + 31) / 32;
    uint32_t* above = ev_smem;                       // one bit per token: its key is above the threshold; later: it stays
    uint32_t* level = above + words;                 // its key is the threshold
    uint32_t* keys = level + words;
    const bool held = n <= p.smem_keys;
    const auto make_key = [&](int t) -> uint32_t {
        const int at_pos = position(t);
        return at_pos < p.sink || at_pos >= seen - p.recent ? 0xffffffffu : evict_key(mass[t]);
    };
    if (held) {
        for (int t = tid; t < n; t += THREADS) keys[t] = make_key(t);
        __syncthreads();
    }
    const auto key_of = [&](int t) { return held ? keys[t] : make_key(t); };

    int turn = 0;
    uint32_t threshold = 0;                          // the largest that at least `keep` keys reach
    for (int shift = 30; shift >= 0; shift -= 2) {
        const uint32_t c1 = threshold + (1u << shift), c2 = threshold + (2u << shift), c3 = threshold + (3u << shift);
        uint32_t n1 = 0, n2 = 0, n3 = 0;
        for (int t = tid; t < n; t += THREADS) {
            const uint32_t k = key_of(t);
            n1 += k >= c1;
            n2 += k >= c2;
            n3 += k >= c3;
        }
        const uint64_t sum = block_sum<THREADS>((uint64_t)n1 | (uint64_t)n2 << 21 | (uint64_t)n3 << 42, buf, turn);
        const auto reach = [&](int i) { return (int)(sum >> (21 * i) & 0x1fffff) >= keep; };
        if (reach(2)) threshold = c3;
        else if (reach(1)) threshold = c2;
        else if (reach(0)) threshold = c1;
    }
    uint32_t over = 0;
    for (int t0 = tid - lane; t0 < words * 32; t0 += THREADS) {
        const int t = t0 + lane;
        const uint32_t k = t < n ? key_of(t) : 0;
        const uint32_t a = __ballot_sync(0xffffffffu, t < n && k > threshold), l = __ballot_sync(0xffffffffu, t < n && k == threshold);
        if (lane == 0) {
            above[t0 / 32] = a;
            level[t0 / 32] = l;
            over += __popc(a);
        }
    }
    const int need = keep - (int)block_sum<THREADS>(over, buf, turn);          // how many at the threshold stay
    // words of a thread: consecutive ones, so that prefix sums over threads go by place
    const int each = (words + THREADS - 1) / THREADS;
    const int w0 = tid * each < words ? tid * each : words, w1 = w0 + each < words ? w0 + each : words;
    uint32_t ties = 0;
    for (int w = w0; w < w1; ++w) ties += __popc(level[w]);
    uint64_t total;
    int left = need - (int)block_prefix<THREADS>(ties, buf, turn, total);      // that the thread's words may still give
    uint32_t holes = 0, movers = 0;
    const auto in_front = [&](int w) { return w * 32 + 32 <= keep ? 0xffffffffu : w * 32 >= keep ? 0u : (1u << (keep - w * 32)) - 1u; };
    for (int w = w0; w < w1; ++w) {
        uint32_t l = level[w], stay = above[w];
        while (l != 0 && left > 0) {                 // the lowest places first
            stay |= l & (0u - l);
            l &= l - 1;
            --left;
        }
        above[w] = stay;
        holes += __popc(~stay & in_front(w));
        movers += __popc(stay & ~in_front(w));
    }
    const uint64_t first = block_prefix<THREADS>((uint64_t)holes | (uint64_t)movers << 32, buf, turn, total);
    int hole = (int)(uint32_t)first, mover = (int)(first >> 32);
    int32_t* from = p.from + unit * p.max_moves;
    int32_t* to = p.to + unit * p.max_moves;
    for (int w = w0; w < w1; ++w) {
        for (uint32_t x = ~above[w] & in_front(w); x != 0; x &= x - 1) to[hole++] = w * 32 + __ffs((int)x) - 1;
        for (uint32_t x = above[w] & ~in_front(w); x != 0; x &= x - 1) from[mover++] = w * 32 + __ffs((int)x) - 1;
    }
    __syncthreads();
    const int moves = (int)(uint32_t)total;
    if (tid == 0) p.count[unit] = moves;
    for (int t = tid; t < keep; t += THREADS)
        if (above[t >> 5] >> (t & 31) & 1u) copy(t);
    for (int i = tid; i < moves; i += THREADS) {
        const int s = from[i], d = to[i];
        p.mass_out[at + d] = mass[s];
        p.pos_out[at + d] = position(s);
    }
}

constexpr int kEvWarps = 8;
constexpr int kEvEach = 4;            // tokens of a warp, their loads in flight together

// CHUNKS: 16-byte pieces of a token's key (as many of its value)
template <int CHUNKS>
__global__ void __launch_bounds__(kEvWarps * 32)
evict_move_kernel(const EvictParams p, int parts) {
    constexpr int kLoads = 2 * CHUNKS / 32;
    wait_for_front();
    const int64_t unit = blockIdx.x / parts;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = ((int)(blockIdx.x % parts) * kEvWarps + warp) * kEvEach;
    const int moves = p.count[unit];
    if (first >= moves) return;
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv);
    const int start = p.kv_indptr[b], first_fill = p.sink_tokens > 0 ? p.sink_tokens : kPageSize;
    uint4* cache = (uint4*)p.cache;
    // the 16-byte piece `c` of the token in place t: its key's, then its value's; -1: no such page
    const auto piece = [&](int t, int c) -> int64_t {
        int e, slot;
        page_of_pos(t, first_fill, e, slot);
        const int64_t page = p.kv_indices[start + e];
        if (page < 0 || page >= p.num_pages) return -1;
        return (((page * 2 + c / CHUNKS) * kPageSize + slot) * p.Hkv + h) * CHUNKS + c % CHUNKS;
    };
    const int n = moves - first < kEvEach ? moves - first : kEvEach;
    uint4 v[kEvEach][kLoads];
    int64_t dst[kEvEach][kLoads];
#pragma unroll
    for (int i = 0; i < kEvEach; ++i) {
        if (i >= n) break;
        const int s = p.from[unit * p.max_moves + first + i], d = p.to[unit * p.max_moves + first + i];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int64_t src = piece(s, j * 32 + lane);
            dst[i][j] = src < 0 ? -1 : piece(d, j * 32 + lane);
            if (dst[i][j] >= 0) v[i][j] = cache[src];
            else report(p.status, KTK_STATUS_BAD_PAGE);
        }
    }
#pragma unroll
    for (int i = 0; i < kEvEach; ++i) {
        if (i >= n) break;
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            if (dst[i][j] >= 0) cache[dst[i][j]] = v[i][j];
    }
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
    const size_t bits = (size_t)((most + 31) / 32) * 2 * sizeof(uint32_t), room = 200 * 1024;
    p.smem_keys = bits + most * sizeof(uint32_t) <= room ? (int)most : 0;
    const size_t smem = bits + (size_t)p.smem_keys * sizeof(uint32_t);
    cudaStream_t st = (cudaStream_t)stream;
    const bool wide = most > 4096;
    const auto kernel = wide ? evict_plan_kernel<1024> : evict_plan_kernel<256>;
    KTK_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), who);
    KTK_CUDA_TRY(launch_behind(false, kernel, (unsigned)units, wide ? 1024 : 256, smem, st, p), who);
    const int parts = (p.max_moves + kEvWarps * kEvEach - 1) / (kEvWarps * kEvEach);
    if (units * parts > 2147483647LL) {
        set_error("%s: too many tokens to move in one launch", who);
        return KTK_ERR_TOO_LARGE;
    }
    if (s->dtype == KTK_F32)
        KTK_CUDA_TRY(launch_behind(true, evict_move_kernel<32>, (unsigned)(units * parts), kEvWarps * 32, 0, st, p, parts), who);
    else
        KTK_CUDA_TRY(launch_behind(true, evict_move_kernel<16>, (unsigned)(units * parts), kEvWarps * 32, 0, st, p, parts), who);
    return KTK_OK;
}
