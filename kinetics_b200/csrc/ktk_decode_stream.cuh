// The balanced partition of page lists over CTAs (ktk_decode_stream.cu): which positions a CTA owns, and which piece of which list
// they are.
#pragma once

#include "ktk_decode_mma.cuh"

namespace ktk {

// Pages: below this a CTA is not worth its start-up.  The form that accumulates weights has a second launch anyway and joins pieces by
// more CTAs: there one page per consumer warp is.
constexpr int kStreamMinChunk = 16, kStreamMinChunkMass = kMmaConsumers;

struct StreamParams {
    DecodeParams d;
    MassParams m;    // read by the kernels that accumulate weights
    int G;
    int min_chunk;   // kStreamMinChunk, or that of the form that accumulates weights
    int wmax;        // padded mode: positions per unit
    int chunk;       // padded mode: positions per CTA
    int64_t total;   // padded mode: units * wmax
    int exact;       // 1: dense CSR lists without a page_count view -- positions are the CSR entries themselves,
                     //    unit (b, h) covers [(indptr[b] - indptr[0]) * Hkv + h * n(b), ... + n(b)), so ragged
                     //    batches are cut evenly too; total and chunk are computed on the device
};

// positions [p0, p1) of CTA c; empty if p1 <= p0
struct Range {
    int64_t p0, p1;
};

// number of positions and positions per CTA, of a decode of `ctas` CTAs
__device__ __forceinline__ void stream_extent(const StreamParams& p, int64_t ctas, int64_t& total, int64_t& chunk) {
    total = p.total;
    chunk = p.chunk;
    if (p.exact) {
        total = (int64_t)(p.d.kv_indptr[p.d.batch] - p.d.kv_indptr[0]) * p.d.Hkv;
        chunk = (total + ctas - 1) / ctas;
        if (chunk < p.min_chunk) chunk = p.min_chunk;
    }
}
__device__ __forceinline__ void stream_extent(const StreamParams& p, int64_t& total, int64_t& chunk) {
    stream_extent(p, gridDim.x, total, chunk);
}

__device__ __forceinline__ Range cta_range(const StreamParams& p, int64_t c) {
    Range r;
    int64_t total, chunk;
    stream_extent(p, total, chunk);
    r.p0 = c * chunk;
    r.p1 = (r.p0 + chunk < total) ? r.p0 + chunk : total;
    return r;
}

// The unit (b, h) whose positions are [start, start + len)
struct Cursor {
    int b, h, len;
    int64_t start;
};

// exact mode: the sequence whose CSR entries contain entry q (relative to indptr[0]); all lanes of the
// warp take part, 32 probes per round
__device__ __forceinline__ int find_sequence(const int32_t* indptr, int B, int64_t q) {
    const int lane = threadIdx.x & 31;
    const int64_t base = indptr[0];
    int lo = 0, hi = B;                                   // invariant: indptr[lo] - base <= q, answer in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int idx = lo + lane * step;
        const bool ok = idx < hi && (int64_t)indptr[idx] - base <= q;
        const unsigned m = __ballot_sync(0xffffffffu, ok);            // a prefix of the lanes: lane 0 always holds
        const int k = 31 - __clz((int)m);
        lo += k * step;
        hi = (lo + step < hi) ? lo + step : hi;
    }
    return lo;
}

__device__ __forceinline__ Cursor cursor_at(const StreamParams& p, int64_t pos) {
    Cursor c;
    if (!p.exact) {
        const int64_t u = pos / p.wmax;
        c.b = (int)(u / p.d.Hkv);
        c.h = (int)(u % p.d.Hkv);
        c.start = u * p.wmax;
        c.len = p.wmax;
        return c;
    }
    const int32_t* ip = p.d.kv_indptr;
    c.b = find_sequence(ip, p.d.batch, pos / p.d.Hkv);
    c.len = ip[c.b + 1] - ip[c.b];
    const int64_t first = (int64_t)(ip[c.b] - ip[0]) * p.d.Hkv;
    c.h = (int)((pos - first) / c.len);
    c.start = first + (int64_t)c.h * c.len;
    return c;
}

__device__ __forceinline__ void cursor_next(const StreamParams& p, Cursor& c) {
    c.start += c.len;
    if (++c.h < p.d.Hkv) return;
    c.h = 0;
    ++c.b;
    if (p.exact) {
        while (c.b < p.d.batch && (c.len = p.d.kv_indptr[c.b + 1] - p.d.kv_indptr[c.b]) == 0) ++c.b;   // no positions
    }
}

// The part of the cursor's unit that falls into the position range [p0, p1).
struct Piece {
    int b, h;
    EntryList el;
    int e_lo, e_hi;   // entries of the unit this CTA runs
    bool first;       // the unit's positions start inside the range
    bool bad;
};

__device__ __forceinline__ Piece get_piece(const StreamParams& p, const Cursor& c, int64_t p0, int64_t p1) {
    Piece pc;
    pc.b = c.b;
    pc.h = c.h;
    pc.el = entry_list(p.d, pc.b, pc.h, pc.bad);
    if (pc.el.cnt > c.len) {          // a list longer than the caller's bound: flagged by the producer, clipped here
        pc.el.cnt = c.len;
        pc.bad = true;
    }
    const int lo = (p0 > c.start) ? (int)(p0 - c.start) : 0;
    const int hi = (p1 - c.start < c.len) ? (int)(p1 - c.start) : c.len;
    pc.first = (p0 <= c.start);
    pc.e_lo = lo < pc.el.cnt ? lo : pc.el.cnt;
    pc.e_hi = hi < pc.el.cnt ? hi : pc.el.cnt;
    return pc;
}

// Behind the MASS form of the decode: merges the pieces of cut lists and adds up the weights (ktk_decode_mass.cu).
int launch_mass_finish(const StreamParams& p, int decode_ctas, cudaStream_t st);

}  // namespace ktk
