// Eviction from a paged cache by accumulated attention weight: of every (sequence, kv head) with more than `keep` tokens the ones
// of largest mass stay, with the first and the newest.  The kept tokens behind place `keep` move into the holes in front of it.
//
// A CTA per (sequence, kv head), or a cluster of them, plans: every token has a 32-bit key whose order is that of the masses (the
// first and newest: the largest key, NaN: the smallest).  The keep-th largest key is found from counts of the keys in intervals; tokens at
// exactly that key stay from the lowest place on.  Which tokens stay is held as one bit
// each, and prefix sums over the bits' words number the holes and the tokens that move.
// Keys and values are copied a warp to a token: behind the plan where few can move or rows are few, else by a launch of their own, whose many
// warps hide the chain of loads (list, page table, cache) that each copy is.
//
// Two copies of a row per token are what an eviction cannot do without: 48 sequences of 2304 tokens cut to 2048, 8 kv heads, 101 MB: the
// copies at 4.8 TB/s (17 us), the plan in front of them 15, most of it the latency of its steps (loads 4, threshold 3, numbers and
// lists 2).
#include <cooperative_groups.h>

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
    int32_t* count;                   // of evict_long_kernel: [units] tokens that move
    int32_t* from;                    // [units][max_moves] their places
    int32_t* to;                      // [units][max_moves] the holes
    int max_moves;
    int32_t* status;
};

constexpr int kEvMaxPages = 32768;

__device__ __forceinline__ uint32_t evict_key(float mass) {
    return mass != mass ? 0u : score_to_key(mass);        // NaN less than -inf (whose key is above 0)
}

// Exclusive prefix sum over the block's threads, and the total.  Two buffers in turn: one barrier each.
template <int THREADS, typename T>
__device__ __forceinline__ T block_prefix(T x, uint64_t (*buf)[32], int& turn, T& total) {
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) buf[turn][warp] = incl;
    __syncthreads();
    const T w = lane < W ? (T)buf[turn][lane] : 0;
    T wi = w;
#pragma unroll
    for (int o = 1; o < W; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, wi, o);
        if (lane >= o) wi += y;
    }
    total = __shfl_sync(0xffffffffu, wi, W - 1);
    turn ^= 1;
    return __shfl_sync(0xffffffffu, wi - w, warp) + incl - x;
}

// A (sequence, kv head) and its tokens; false: nothing is evicted from it
struct EvictUnit {
    int n, stored, seen, start, first_fill;
    int64_t at;                                      // of its row in masses and positions
    const float* mass;
    const int32_t* pos;
    // both loads are always made, so that those of several tokens can be in flight together
    __device__ __forceinline__ int position(int t) const {
        const int at = pos[t < stored ? t : 0];
        return t < stored ? at : seen - n + t;
    }
};
__device__ __forceinline__ bool evict_unit(const EvictParams& p, int64_t unit, int most, EvictUnit& u) {
    const int b = (int)(unit / p.Hkv), h = (int)(unit % p.Hkv);
    const SeqPages sp = seq_pages(p.kv_indptr, p.page_count, p.kv_last_page_len, p.sink_tokens, b);
    const int row = p.slot_index ? p.slot_index[b] : b;
    u.n = sp.total;
    u.start = sp.start;
    u.first_fill = sp.first_fill;
    if (u.n <= 0 && !sp.bad) return false;           // an idle row: its slot may be none
    if (sp.bad || row < 0 || row >= p.rows || u.n > p.stride || sp.n_pages > p.max_pages || u.n > most) {
        if (threadIdx.x == 0) report(p.status, KTK_STATUS_BAD_TABLE);
        return false;
    }
    u.at = ((int64_t)row * p.Hkv + h) * p.stride;
    u.mass = p.mass_in + u.at;
    u.pos = p.pos_in + u.at;
    u.stored = p.stored[row];
    u.seen = p.seen[row];
    return true;
}
// What a token in front of place `keep` has if it stays; holes are written over later.  The key of a token.
struct EvictToken {
    float mass;
    int pos;
};
__device__ __forceinline__ EvictToken read_token(const EvictUnit& u, int t) { return {u.mass[t], u.position(t)}; }
__device__ __forceinline__ void keep_token(const EvictParams& p, const EvictUnit& u, int t, const EvictToken& x) {
    if (p.mass_in != p.mass_out) p.mass_out[u.at + t] = x.mass;
    if (p.pos_in != p.pos_out || t >= u.stored) p.pos_out[u.at + t] = x.pos;
}
__device__ __forceinline__ uint32_t key_of(const EvictParams& p, const EvictUnit& u, const EvictToken& x) {
    return x.pos < p.sink || x.pos >= u.seen - p.recent ? 0xffffffffu : evict_key(x.mass);
}

// The words of places in front of `keep`
__device__ __forceinline__ uint32_t in_front(int w, int keep) {
    return w * 32 + 32 <= keep ? 0xffffffffu : w * 32 >= keep ? 0u : (1u << (keep - w * 32)) - 1u;
}

// The CTAs of a cluster, and an array that each of them has
struct Cluster {
    int size, rank;
    __device__ __forceinline__ void sync() const {
        if (size > 1) cooperative_groups::this_cluster().sync();
        else __syncthreads();
    }
    template <typename T> __device__ __forceinline__ const T* of(const T* mine, int r) const {
        return size > 1 ? cooperative_groups::this_cluster().map_shared_rank(mine, r) : mine;
    }
};

// The keep-th largest key and how many keys are above it.  walk(visit): calls visit(key, there) for the CTA's keys, whole warps together.
// Counts of the keys in equal intervals from the smallest positive mass to the largest say in which it lies; up to kEvRanked keys there
// are ranked directly, more are counted in intervals of that interval.  (Intervals of all 32-bit keys, which hold masses of a few
// octaves in a dozen of them, took three rounds.)  All CTAs of the cluster find the same.
constexpr int kEvRanked = 256;
constexpr uint32_t kEvSafe = 0xffffffffu, kEvZero = 0x80000000u;        // keys of the first and newest tokens, and of a mass of 0
struct Threshold {
    uint32_t key;
    int above;
};
template <int THREADS> struct ThresholdShared {
    static constexpr int kBins = 2 * THREADS;         // a power of two; two of them to a thread
    uint32_t hist[2][kBins];                          // begin as zeros; one, then the other half of a warp counts there
    uint32_t some[kEvRanked], all[kEvRanked];
    uint32_t found[3], count;                        // count begins as 0
    uint4 range;
};
template <int THREADS> __device__ __forceinline__ void clear_counts(ThresholdShared<THREADS>& sh) {
    reinterpret_cast<uint4*>(sh.hist[0])[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
    if (threadIdx.x == 0) sh.count = 0;
}
template <int THREADS, class Walk>
__device__ __forceinline__ Threshold find_threshold(int keep, const Cluster& cl, ThresholdShared<THREADS>& sh, uint64_t (*buf)[32], int& turn, Walk walk) {
    static_assert(kEvRanked <= THREADS, "a thread to a ranked key");
    constexpr int kBins = ThresholdShared<THREADS>::kBins, kLog = THREADS == 256 ? 9 : 11, W = THREADS / 32;
    static_assert(kBins == 1 << kLog, "intervals by shifts");
    const int tid = threadIdx.x, lane = tid & 31;
    // smallest and largest key of the positive masses, and of the others
    uint32_t lo = kEvSafe, hi = 0, low = kEvSafe, high = 0;
    walk([&](uint32_t key, bool on) {
        const bool positive = key > kEvZero;
        if (on && positive && key != kEvSafe) {
            lo = min(lo, key);
            hi = max(hi, key);
        }
        if (on && !positive) {
            low = min(low, key);
            high = max(high, key);
        }
    });
    const auto reduce = [&] {
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
    };
    reduce();
    uint4* ranges = reinterpret_cast<uint4*>(sh.all);            // of the warps
    if (lane == 0) ranges[tid >> 5] = make_uint4(lo, hi, low, high);
    __syncthreads();
    const auto take = [&](const uint4* from) {
        const uint4 x = *from;
        lo = x.x, hi = x.y, low = x.z, high = x.w;
        reduce();
    };
    take(ranges + (lane < W ? lane : 0));
    if (cl.size > 1) {
        if (tid == 0) sh.range = make_uint4(lo, hi, low, high);
        cl.sync();
        take(cl.of(&sh.range, lane < cl.size ? lane : 0));
    }
    // The keys in question: base .. base + span.  In round 0 all of them: interval 0 is that of masses that are not positive, the last that
    // of kEvSafe.
    Threshold r{0, 0};
    uint32_t base = lo, span = lo < hi ? hi - lo : 0;
    const auto inside = [&](uint32_t key) { return key - base <= span; };
    for (int round = 0; ; ++round) {
        int shift = max(32 - kLog - __clz(span | 1u), 0);
        if (round == 0) {
            if (span >> shift > kBins - 3) ++shift;
            uint32_t* copy = sh.hist[lane >> 4];
            walk([&](uint32_t key, bool on) {
                if (on) atomicAdd(&copy[key == kEvSafe ? kBins - 1 : key < base ? 0 : 1 + ((key - base) >> shift)], 1u);
            });
        } else {
            if (cl.size > 1) {                       // zeros again, when all have read
                cl.sync();
                sh.hist[0][tid] = sh.hist[0][tid + THREADS] = 0;
                __syncthreads();
            }
            walk([&](uint32_t key, bool on) {
                on = on && inside(key);
                const unsigned active = __ballot_sync(0xffffffffu, on);
                if (active == 0) return;
                // a warp whose keys share an interval (the same mass) adds once
                const uint32_t bin = (key - base) >> shift, one = __shfl_sync(0xffffffffu, bin, __ffs((int)active) - 1);
                if (__all_sync(0xffffffffu, !on || bin == one)) {
                    if (lane == 0) atomicAdd(&sh.hist[0][one], (uint32_t)__popc(active));
                } else if (on) {
                    atomicAdd(&sh.hist[0][bin], 1u);
                }
            });
        }
        if (cl.size > 1) {                           // sums over the CTAs to the second array
            if (round == 0) {
                __syncthreads();
                for (int i = tid; i < kBins; i += THREADS) sh.hist[0][i] += sh.hist[1][i];
            }
            cl.sync();
            uint32_t sums[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < cl.size)
#pragma unroll
                    for (int k = 0; k < 2; ++k) sums[k] += cl.of(sh.hist[0], i)[k * THREADS + tid];
            sh.hist[1][tid] = sums[0];
            sh.hist[1][tid + THREADS] = sums[1];
        }
        __syncthreads();
        // from the largest interval on, two to a thread, which leaves zeros
        const int bin0 = kBins - (tid + 1) * 2;
        uint2* at = reinterpret_cast<uint2*>(&sh.hist[1][bin0]);
        uint2 c = *at;
        *at = make_uint2(0u, 0u);
        if (cl.size == 1) {
            at = reinterpret_cast<uint2*>(&sh.hist[0][bin0]);
            c.x += at->x;
            c.y += at->y;
            *at = make_uint2(0u, 0u);
        }
        uint32_t total;
        const uint32_t sum = c.x + c.y;
        uint32_t need = (uint32_t)(keep - r.above);
        const uint32_t before = block_prefix<THREADS>(sum, buf, turn, total);
        if (before < need && need <= before + sum) {             // one thread
            const bool upper = need <= before + c.y;
            sh.found[0] = (uint32_t)(bin0 + (upper ? 1 : 0));
            sh.found[1] = upper ? before : before + c.y;
            sh.found[2] = upper ? c.y : c.x;
        }
        __syncthreads();
        const uint32_t bin = sh.found[0], here = sh.found[2];
        r.above += (int)sh.found[1];
        need -= sh.found[1];
        if (round > 0) {
            base += bin << shift;
            span = (1u << shift) - 1u;
        } else if (bin == kBins - 1) {
            return {kEvSafe, 0};                     // as many first and newest ones as stay
        } else if (bin > 0) {
            base += (bin - 1) << shift;
            span = (1u << shift) - 1u;
        } else {
            base = low;
            span = high - low;
        }
        if (here == need) return {base - 1, keep};   // all of the interval stay; it is not that from 0 on: there are more than `keep` keys
        if (span == 0) return {base, r.above};
        if (here <= kEvRanked) {
            uint32_t put = 0;                        // of the warp's keys, the first one's place
            walk([&](uint32_t key, bool on) { put += __popc(__ballot_sync(0xffffffffu, on && inside(key))); });
            if (lane == 0 && put > 0) put = atomicAdd(&sh.count, put);
            put = __shfl_sync(0xffffffffu, put, 0);
            walk([&](uint32_t key, bool on) {
                on = on && inside(key);
                const unsigned active = __ballot_sync(0xffffffffu, on);
                if (on) sh.some[put + __popc(active & ((1u << lane) - 1u))] = key;
                put += __popc(active);
            });
            if (tid < kEvRanked) sh.all[tid] = 0;
            cl.sync();
            if (tid < (int)here) {
                int i = 0, at = tid;                 // the tid-th of the CTAs' keys, one CTA's behind the other's
                for (; i + 1 < cl.size; ++i) {
                    const int n = (int)*cl.of(&sh.count, i);
                    if (at < n) break;
                    at -= n;
                }
                sh.all[tid] = cl.of(sh.some, i)[at];
            }
            __syncthreads();
            if (tid < (int)here) {
                const uint32_t key = sh.all[tid];
                uint32_t greater = 0, equal = 0;     // the zeros behind the last are equal to the smallest key at most
#pragma unroll 4
                for (uint32_t i = 0; i < here; i += 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(sh.all + i);
                    greater += (v.x > key) + (v.y > key) + (v.z > key) + (v.w > key);
                    equal += (v.x == key) + (v.y == key) + (v.z == key) + (v.w == key);
                }
                if (greater < need && need <= greater + equal) {                 // all that do hold the same key
                    const bool stay = need == greater + equal;                   // all of that key do
                    sh.found[0] = stay ? key - 1 : key;
                    sh.found[1] = (uint32_t)(stay ? keep : r.above + (int)greater);
                }
            }
            __syncthreads();
            return {sh.found[0], (int)sh.found[1]};
        }
        __syncthreads();                             // found may be written again
    }
}

// The CTA's words of stay, level: one bit per token, its key is above the threshold, at it; `need` of the latter, over the cluster,
// stay.  Afterwards `stay` says which tokens stay and `level` holds, for words in front of place `keep`, the holes in words before, for
// those behind the tokens that move.  first: number of the CTA's first word; shared: two words that the cluster's CTAs read of each
// other.  Returns how many tokens of the cluster move.
template <int THREADS>
__device__ __forceinline__ int number_moves(uint32_t* stay, uint32_t* level, int first, int words, int keep, int need, const Cluster& cl,
                                            uint64_t* shared, uint64_t (*buf)[32], int& turn) {
    const int tid = threadIdx.x;
    // words of a thread: consecutive ones, so that prefix sums over threads go by place
    const int each = (words + THREADS - 1) / THREADS;
    const int w0 = tid * each < words ? tid * each : words, w1 = w0 + each < words ? w0 + each : words;
    // sums over the CTAs in front, and over all
    const auto over_cluster = [&](uint64_t* mine, uint64_t total, uint64_t& all) -> uint64_t {
        if (cl.size == 1) {
            all = total;
            return 0;
        }
        if (tid == 0) *mine = total;
        cl.sync();
        uint64_t before = 0;
        all = 0;
        for (int i = 0; i < cl.size; ++i) {
            const uint64_t x = *cl.of(mine, i);
            if (i < cl.rank) before += x;
            all += x;
        }
        return before;
    };
    uint64_t all, total;
    if (need > 0) {
        uint64_t ties = 0;
        for (int w = w0; w < w1; ++w) ties += __popc(level[w]);
        const uint64_t before = block_prefix<THREADS>(ties, buf, turn, total);
        int left = need - (int)(before + over_cluster(&shared[0], total, all));
        for (int w = w0; w < w1; ++w) {
            uint32_t l = level[w], more = 0;
            if (left >= __popc(l)) {
                more = l;
                left -= __popc(l);
            } else {
                for (; left > 0; l &= l - 1, --left) more |= l & (0u - l);       // the lowest places first
            }
            stay[w] |= more;
        }
    }
    uint64_t count = 0;                              // holes | tokens that move
    const auto add = [&](int w) {
        count += (uint64_t)__popc(~stay[w] & in_front(first + w, keep)) | (uint64_t)__popc(stay[w] & ~in_front(first + w, keep)) << 32;
    };
    for (int w = w0; w < w1; ++w) add(w);
    count = block_prefix<THREADS>(count, buf, turn, total);
    count += over_cluster(&shared[1], total, all);
    for (int w = w0; w < w1; ++w) {
        level[w] = (first + w) * 32 < keep ? (uint32_t)count : (uint32_t)(count >> 32);
        add(w);
    }
    return (int)(uint32_t)all;
}
// What becomes of the token in place t: hole(i) the i-th hole is there, mover(i) it is the i-th token that moves
template <class Hole, class Mover>
__device__ __forceinline__ void token_move(const uint32_t* stay, const uint32_t* level, int first, int t, int keep, Hole hole, Mover mover) {
    const int w = t >> 5;
    const uint32_t s = stay[w - first], bit = 1u << (t & 31), below = bit - 1;
    if (t < keep) {
        if (!(s & bit)) hole((int)level[w - first] + __popc(~s & below));
    } else if (s & bit) {
        const uint32_t front = in_front(w, keep);
        mover((front ? 0 : (int)level[w - first]) + __popc(s & below & ~front));         // only words in front lie before one that is cut
    }
}

// Copies keys and values of moves first .. first + EACH - 1 (of `moves`): from(i) -> to(i), by a whole warp, their loads in flight
// together.  Two lanes find where a move leads, all lanes then copy.  CHUNKS: 16-byte pieces of a token's key (as many of its value)
template <int CHUNKS, int EACH, class From, class To>
__device__ __forceinline__ void copy_tokens(const EvictParams& p, int h, int start, int first_fill, int first, int moves, From from, To to) {
    constexpr int kLoads = 2 * CHUNKS / 32;
    const int lane = threadIdx.x & 31;
    uint4* cache = (uint4*)p.cache;
    int64_t at = -1;                                 // first piece of the token's key; -1: no such page
    const int move = first + lane / 2;
    if (lane < 2 * EACH && move < moves) {
        int e, slot;
        page_of_pos(lane % 2 ? to(move) : from(move), first_fill, e, slot);
        const int64_t page = __ldg(p.kv_indices + start + e);
        if (page < 0 || page >= p.num_pages) report(p.status, KTK_STATUS_BAD_PAGE);
        else at = ((page * 2 * kPageSize + slot) * p.Hkv + h) * CHUNKS;
    }
    const int64_t to_value = (int64_t)kPageSize * p.Hkv * CHUNKS;                // from a token's key to its value
    int64_t mine[kLoads];                            // this lane's pieces from the first on
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int c = j * 32 + lane;
        mine[j] = c < CHUNKS ? c : to_value + c - CHUNKS;
    }
    uint4 v[EACH][kLoads];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int64_t src = __shfl_sync(0xffffffffu, at, 2 * i);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            if (src >= 0) v[i][j] = cache[src + mine[j]];
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int64_t src = __shfl_sync(0xffffffffu, at, 2 * i), dst = __shfl_sync(0xffffffffu, at, 2 * i + 1);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            if (src >= 0 && dst >= 0) cache[dst + mine[j]] = v[i][j];
    }
}

// Tokens that are copied behind the plan, in the same launch, where few rows leave SMs for more CTAs that copy (up to kEvCopiers a row) or few
// tokens move; more go to a launch of their own, which costs the host 3 us and a workspace.  Replayed from a graph / called, one launch
// and two, 8 kv heads, sequences of 2048 + 256 tokens cut to 2048: one, 8 copiers, 9.8 / 12.8 us and 11.3 / 16.3; four, 4 copiers, 12.3 / 12.8 and
// 11.6 / 16.6; eight, 2 copiers, 14.9 / 15.6 and 12.4 / 16.4; seven fp32 ones of 150 to 701 cut to 333, 4 kv heads, 4 copiers, 10.1 / 11.0 and
// 9.7 / 16.0; 48 of 2048 + 128, one copier, 25.8 / 27.0 and 27.2 / 29.1.
constexpr int kEvFused = 128, kEvFusedEach = 96, kEvCopiers = 8;

// Sequences of at most THREADS * ITEMS tokens per CTA, keys in registers.  CHUNKS == 0: a cluster plans, keys and values are left to
// evict_move_kernel.  Else CHUNKS is the number of 16-byte pieces of a token's key: one CTA plans, and with the others of its cluster, the
// `copiers`, copies from the lists in its shared memory.
template <int THREADS, int ITEMS, int CHUNKS>
__global__ void __launch_bounds__(THREADS)
evict_kernel(const EvictParams p, int cluster, int copiers) {
    constexpr int kMost = THREADS * ITEMS, kWords = kMost / 32;
    // tokens of a thread whose loads are in flight together: of 256 threads 12 (48 sequences of 2304 tokens 31.9 us, 32.9
    // with 8; 100 of 150 to 701 21.9 us, 23.2 with 16); 1024 threads have registers for 8
    constexpr int kBatch = THREADS == 256 ? 12 : 8;
    __shared__ uint64_t buf[2][32], shared[2];
    __shared__ __align__(16) ThresholdShared<THREADS> counts;
    __shared__ uint32_t stay[kWords], level[kWords];
    const int tid = threadIdx.x;
    clear_counts<THREADS>(counts);
    wait_for_front();
    const int copier = CHUNKS > 0 ? (int)(blockIdx.x % copiers) : 0;
    const Cluster cl = CHUNKS > 0 ? Cluster{1, 0} : Cluster{cluster, (int)(blockIdx.x % cluster)};
    const int64_t unit = blockIdx.x / (CHUNKS > 0 ? copiers : cluster);
    EvictUnit u;
    const bool there = evict_unit(p, unit, kMost * cl.size, u);                  // the same for the cluster
    if (CHUNKS == 0 && (!there || u.n <= p.keep) && tid == 0) p.count[unit] = 0;
    if (!there) return;
    const int keep = p.keep, front = u.n < keep ? u.n : keep;
    // the CTA's tokens: whole words
    const int words = ((u.n + 31) / 32 + cl.size - 1) / cl.size, first = cl.rank * words, t0 = first * 32;
    const int n = min(u.n - t0, words * 32);         // may be negative
    extern __shared__ int32_t ev_list[];             // of CTAs that copy
    int32_t *from = CHUNKS > 0 ? ev_list : p.from + unit * p.max_moves, *to = CHUNKS > 0 ? ev_list + p.max_moves : p.to + unit * p.max_moves;
    __shared__ int planned;
    int moves = 0;
    if (copier > 0) {
        if (u.n <= keep) return;
    } else {
        uint32_t key[ITEMS];
#pragma unroll
        for (int j0 = 0; j0 < ITEMS; j0 += kBatch) {     // reads of a batch, then its writes
            if (j0 * THREADS >= n) break;
            EvictToken x[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch && j0 + j < ITEMS; ++j) x[j] = read_token(u, min(t0 + (j0 + j) * THREADS + tid, u.n - 1));
#pragma unroll
            for (int j = 0; j < kBatch && j0 + j < ITEMS; ++j) {
                const int i = (j0 + j) * THREADS + tid;
                key[j0 + j] = key_of(p, u, x[j]);
                if (i < n && t0 + i < front) keep_token(p, u, t0 + i, x[j]);
            }
        }
        if (u.n <= keep) return;
        __syncthreads();
        const auto each_item = [&](auto visit) {         // of the CTA's tokens, whole warps
#pragma unroll
            for (int j = 0; j < ITEMS; ++j) {
                if (j * THREADS >= n) break;             // uniform
                visit(j, j * THREADS + tid);
            }
        };
        int turn = 0;
        const Threshold at = find_threshold<THREADS>(keep, cl, counts, buf, turn, [&](auto visit) {
            each_item([&](int j, int i) { visit(key[j], i < n); });
        });
        each_item([&](int j, int i) {
            const uint32_t a = __ballot_sync(0xffffffffu, i < n && key[j] > at.key), l = __ballot_sync(0xffffffffu, i < n && key[j] == at.key);
            if ((tid & 31) == 0) {
                stay[i / 32] = a;
                level[i / 32] = l;
            }
        });
        __syncthreads();
        moves = number_moves<THREADS>(stay, level, first, n > 0 ? (n + 31) / 32 : 0, keep, keep - at.above, cl, shared, buf, turn);
        __syncthreads();
        each_item([&](int, int i) {
            if (i < n) token_move(stay, level, first, t0 + i, keep, [&](int k) { to[k] = t0 + i; }, [&](int k) { from[k] = t0 + i; });
        });
    }
    if constexpr (CHUNKS > 0) {
        constexpr int W = THREADS / 32, kEach = 4;   // eight took the planning's registers: 64 tokens of 384 CTAs 23.3 us, 20.4
        const int32_t *source = from, *hole = to;    // the planning CTA's
        if (copiers > 1) {
            if (tid == 0) planned = moves;
            auto all = cooperative_groups::this_cluster();
            all.sync();
            moves = *all.map_shared_rank(&planned, 0);
            source = all.map_shared_rank(from, 0);
            hole = all.map_shared_rank(to, 0);
        } else {
            __syncthreads();
        }
        for (int i = (copier * W + (tid >> 5)) * kEach; i < moves; i += copiers * W * kEach)
            copy_tokens<CHUNKS, kEach>(p, (int)(unit % p.Hkv), u.start, u.first_fill, i, moves, [&](int k) { return source[k]; },
                                       [&](int k) { return hole[k]; });
    } else {
        cl.sync();
        if (cl.rank == 0 && tid == 0) p.count[unit] = moves;
    }
    if (copier == 0) {
        for (int i = cl.rank * THREADS + tid; i < moves; i += cl.size * THREADS) {
            const EvictToken x = read_token(u, from[i]);
            p.mass_out[u.at + to[i]] = x.mass;
            p.pos_out[u.at + to[i]] = x.pos;
        }
    }
    if (CHUNKS > 0 && copiers > 1) cooperative_groups::this_cluster().sync();    // the lists are read until here
}

// Longer ones, whose keys fit neither registers nor shared memory: they are made again in every pass.
constexpr int kEvLong = 1024;
__global__ void __launch_bounds__(kEvLong)
evict_long_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t ev_smem[];
    __shared__ uint64_t buf[2][32];
    __shared__ __align__(16) ThresholdShared<kEvLong> counts;
    const int tid = threadIdx.x, lane = tid & 31;
    const Cluster alone{1, 0};
    clear_counts<kEvLong>(counts);
    wait_for_front();
    const int64_t unit = blockIdx.x;
    EvictUnit u;
    if (!evict_unit(p, unit, kEvMaxPages * kPageSize, u)) {
        if (tid == 0) p.count[unit] = 0;
        return;
    }
    const int n = u.n, keep = p.keep, words = (n + 31) / 32;
    uint32_t *stay = ev_smem, *level = stay + words;
    for (int t = tid; t < min(n, keep); t += kEvLong) keep_token(p, u, t, read_token(u, t));
    if (n <= keep) {
        if (tid == 0) p.count[unit] = 0;
        return;
    }
    __syncthreads();
    // a key made again may not see what was written: positions behind `stored` are not read, and masses in place are not written
    const auto each = [&](auto visit) {
        for (int t0 = tid - lane; t0 < n; t0 += kEvLong) {
            const int t = t0 + lane;
            visit(t, t >= n ? 0 : key_of(p, u, read_token(u, t)));
        }
    };
    int turn = 0;
    const Threshold at = find_threshold<kEvLong>(keep, alone, counts, buf, turn, [&](auto visit) {
        each([&](int t, uint32_t key) { visit(key, t < n); });
    });
    each([&](int t, uint32_t key) {
        const uint32_t a = __ballot_sync(0xffffffffu, t < n && key > at.key), l = __ballot_sync(0xffffffffu, t < n && key == at.key);
        if (lane == 0) {
            stay[t / 32] = a;
            level[t / 32] = l;
        }
    });
    __syncthreads();
    const int moves = number_moves<kEvLong>(stay, level, 0, words, keep, keep - at.above, alone, nullptr, buf, turn);
    __syncthreads();
    int32_t *from = p.from + unit * p.max_moves, *to = p.to + unit * p.max_moves;
    for (int t = tid; t < n; t += kEvLong)
        token_move(stay, level, 0, t, keep, [&](int i) { to[i] = t; }, [&](int i) { from[i] = t; });
    __syncthreads();
    if (tid == 0) p.count[unit] = moves;
    for (int i = tid; i < moves; i += kEvLong) {
        const EvictToken x = read_token(u, from[i]);
        p.mass_out[u.at + to[i]] = x.mass;
        p.pos_out[u.at + to[i]] = x.pos;
    }
}
// 16 sequences of 2304 tokens cut to 2048: 17.6 us, 19.3 with four tokens of a warp in flight; CTAs of eight warps leave longer tails (100 fp32
// sequences of 150 to 701 cut to 333: 25.0 us, 22.7).
constexpr int kEvWarps = 4, kEvEach = 8;
template <int CHUNKS>
__global__ void __launch_bounds__(kEvWarps * 32)
evict_move_kernel(const EvictParams p, int parts) {
    wait_for_front();
    const int64_t unit = blockIdx.x / parts;
    const int first = ((int)(blockIdx.x % parts) * kEvWarps + (threadIdx.x >> 5)) * kEvEach;
    const int moves = p.count[unit];
    if (first >= moves) return;
    const int32_t *from = p.from + unit * p.max_moves, *to = p.to + unit * p.max_moves;
    copy_tokens<CHUNKS, kEvEach>(p, (int)(unit % p.Hkv), p.kv_indptr[unit / p.Hkv], p.sink_tokens > 0 ? p.sink_tokens : kPageSize, first, moves,
                        [&](int k) { return from[k]; }, [&](int k) { return to[k]; });
}

// How an eviction is cut, by the caller's bounds
struct EvictCut {
    int64_t units, most, max_moves;
    int cluster;                      // CTAs that plan a unit
    int copiers;                      // CTAs that copy behind the plan, from lists in shared memory
    bool fused;                       // they do; else a launch of its own
    size_t bytes;
};
template <int THREADS, int ITEMS>
static cudaError_t launch_evict(const EvictParams& p, const EvictCut& cut, bool f32, cudaStream_t st) {
    const auto kernel = !cut.fused ? evict_kernel<THREADS, ITEMS, 0> : f32 ? evict_kernel<THREADS, ITEMS, 32> : evict_kernel<THREADS, ITEMS, 16>;
    const size_t smem = cut.fused ? 2 * (size_t)p.max_moves * sizeof(int32_t) : 0;
    const int ctas = cut.fused ? cut.copiers : cut.cluster;
    // Not early are small CTAs in front of a launch of copies, whose CTAs would wait among them (8 sequences of 2304 cut to 2048 13.9 us, 12.4);
    // of the large ones (8 of 16384 cut to 2048) early saves a call 43.2 us -> 40.5.
    const bool early = (cut.fused || THREADS == 1024) && cut.units * ctas <= sm_count();
    return launch_cluster(early, kernel, (unsigned)(cut.units * ctas), THREADS, smem, ctas, st, p, cut.cluster, cut.copiers);
}

static int64_t evict_max_moves(int max_pages, int keep) {
    const int64_t behind = (int64_t)max_pages * kPageSize - keep;
    return behind < 1 ? 1 : behind < keep ? behind : keep;
}

// CTAs per (sequence, kv head): more than one for long sequences where SMs would idle.  Two sequences of 32768 tokens, 8 kv heads, the
// plan alone: 24.4 us with two CTAs of 1024 threads each, 19.0 with four.
static int evict_cluster(int64_t units, int64_t most) {
    int c = 1;
    while (c < 4 && most > 4096 * c && units * c * 2 <= sm_count()) c *= 2;
    return most > 16384 * c ? 4 : c;
}
static EvictCut evict_cut(const ktk_shape* s, int max_pages, int keep) {
    EvictCut c;
    c.units = (int64_t)s->batch * s->num_kv_heads;
    c.most = (int64_t)max_pages * kPageSize;
    c.max_moves = evict_max_moves(max_pages, keep);
    c.cluster = evict_cluster(c.units, c.most);
    c.copiers = 1;
    if (c.cluster == 1)
        while (c.copiers < kEvCopiers && c.max_moves > 32 * c.copiers && c.units * c.copiers * 2 <= sm_count()) c.copiers *= 2;
    c.fused = c.cluster == 1 && (c.max_moves <= kEvFused || c.max_moves <= kEvFusedEach * c.copiers);
    c.bytes = c.fused ? 0 : (size_t)c.units * (1 + 2 * (size_t)c.max_moves) * sizeof(int32_t);
    return c;
}

}  // namespace ktk

using namespace ktk;

extern "C" size_t ktk_evict_workspace_bytes(const ktk_shape* shape, int32_t max_pages_per_seq, int32_t keep) {
    if (check_shape(shape, "ktk_evict_workspace_bytes") != KTK_OK || shape->batch == 0 || keep < 1 || max_pages_per_seq < 1 ||
        max_pages_per_seq > kEvMaxPages)
        return 0;
    return evict_cut(shape, max_pages_per_seq, keep).bytes;
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
    const EvictCut cut = evict_cut(s, max_pages_per_seq, keep);
    const int64_t parts = (cut.max_moves + kEvWarps * kEvEach - 1) / (kEvWarps * kEvEach);
    if (max_pages_per_seq > kEvMaxPages || cut.units * (parts > 8 ? parts : 8) > 2147483647LL) {
        set_error("%s: %d pages per sequence (at most %d), %lld rows", who, max_pages_per_seq, kEvMaxPages, (long long)cut.units);
        return KTK_ERR_TOO_LARGE;
    }
    if (cut.bytes > 0 && (workspace == nullptr || workspace_bytes < cut.bytes)) {
        set_error("%s: workspace of %zu bytes needed, got %zu", who, cut.bytes, workspace ? workspace_bytes : (size_t)0);
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
    p.max_moves = (int)cut.max_moves;
    p.count = (int32_t*)workspace;
    p.from = p.count + cut.units;
    p.to = p.from + cut.units * p.max_moves;

    cudaStream_t st = (cudaStream_t)stream;
    const bool f32 = s->dtype == KTK_F32;
    if (cut.most <= 4096) {
        KTK_CUDA_TRY((launch_evict<256, 16>(p, cut, f32, st)), who);
    } else if (cut.most <= 16384 * cut.cluster) {
        KTK_CUDA_TRY((launch_evict<1024, 16>(p, cut, f32, st)), who);
    } else {
        const size_t smem = (size_t)((cut.most + 31) / 32) * 2 * sizeof(uint32_t);
        KTK_CUDA_TRY(allow_shared(evict_long_kernel, smem), who);
        KTK_CUDA_TRY(launch_behind(false, evict_long_kernel, (unsigned)cut.units, kEvLong, smem, st, p), who);
    }
    if (cut.fused) return KTK_OK;
    const auto move = f32 ? evict_move_kernel<32> : evict_move_kernel<16>;
    KTK_CUDA_TRY(launch_behind(true, move, (unsigned)(cut.units * parts), kEvWarps * 32, 0, st, p, (int)parts), who);
    return KTK_OK;
}
