// paged_sched.cuh -- how the paged attention's work is shared out among the CTAs.
//
// The query rows of one sequence and kv head (its new tokens times the heads that share
// the kv head: row r is token r / group, head r % group) are cut into tiles of kRows
// rows, and the positions that a tile sees into blocks of kBlock.  A unit is one block of
// one tile of one kv head.  The units are numbered kv head by kv head, sequence by
// sequence, tile by tile, block by block, and CTA c of C takes units [U c / C, U (c+1) /
// C): equal shares whatever the lengths are, known on the GPU alone.  A tile that falls
// into several shares is computed in parts (its running max, sum and unnormalised
// output), which paged_join_kernel adds up afterwards, in CTA order.  Every CTA finds its
// share itself: one scan over the sequences' tiles and one over the tiles' units.
#pragma once

#include "common.cuh"
#include "paged.h"
#include "tc_ptx.cuh"

namespace rbt {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^x of the special-function unit (relative error 2^-22; below 2^-126 it gives 0)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr long long kWaitClocks = 4000000000ll;  // 2 s and more: far beyond any legitimate wait

// A wait that gives up once, for good: the softmax then passes its other barriers at once.
struct Waiter {
    bool ok = true;
    unsigned* status;
    __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) {
        if (!ok || tc::mbar_try_wait(bar, parity)) return;
        const long long t0 = clock64();
        while (!tc::mbar_try_wait(bar, parity))
            if (clock64() - t0 > kWaitClocks) {
                ok = false;
                atomicCAS(status, 0u, (unsigned)kPagedWait);
                return;
            }
    }
    __device__ __forceinline__ bool one(uint64_t* bar, uint32_t parity) {
        (*this)(bar, parity);
        return ok;
    }
    // for a whole warp, which goes on only if every lane may
    __device__ __forceinline__ bool warp(uint64_t* bar, uint32_t parity) {
        (*this)(bar, parity);
        return ok = __all_sync(FULL_MASK, ok);
    }
};

struct Seq {
    int row0, count, len;  // first row, new tokens, positions; count 0: not of this launch
};

// Sequence i, checked; what its lengths do not allow leaves a code and no rows.
__device__ __forceinline__ Seq load_seq(const PagedAttnArgs& a, int i) {
    Seq s;
    s.row0 = a.cu[i];
    const int end = a.cu[i + 1];
    s.len = a.len[i];
    s.count = end - s.row0;
    unsigned bad = 0;
    if (s.row0 < 0 || end < s.row0 || end > a.n_rows) bad = kPagedCu;
    else if (s.len < 0 || (long long)s.len > ((long long)a.table_stride << a.page_shift)) bad = kPagedLen;
    if (bad) {
        atomicCAS(a.status, 0u, bad);
        s.count = 0;
    }
    const long long rows = (long long)s.count * a.group;
    if (rows <= a.rows_lo || rows > a.rows_hi) s.count = 0;
    return s;
}

struct Tile {
    int seq, kvh;
    Seq s;
    int r0, rows;    // packed rows [r0, r0 + rows) of the sequence
    int lo, hi;      // positions that some row of the tile sees
    int b0, nb;      // blocks b0 .. b0 + nb
    int off;         // position of a token minus its index: len - count
};

template <int kRows, int kBlock>
__device__ __forceinline__ void tile_range(const PagedAttnArgs& a, const Seq& s, int r0, Tile& t) {
    t.s = s;
    t.r0 = r0;
    t.rows = min(kRows, s.count * a.group - r0);
    t.off = s.len - s.count;
    t.lo = 0;
    t.hi = s.len;
    if (a.causal) {
        t.hi = max(0, min(s.len, t.off + (r0 + t.rows - 1) / a.group + 1));
        if (a.window) t.lo = max(0, t.off + r0 / a.group - a.window + 1);
    }
    t.b0 = t.lo / kBlock;
    t.nb = max(1, (t.hi + kBlock - 1) / kBlock - t.b0);  // a tile that sees nothing is one unit, which writes its zeros
}

// The share of this CTA: `left` units from block `skip` of tile `tile` of kv head `kvh`.
struct Share {
    int tile, kvh, skip;  // index of the tile among one kv head's tiles
    int n_tiles;
    int ctas;             // CTAs with any work
    long long units;      // of all kv heads
    long long left;
};

// largest i with start[i] <= x
__device__ __forceinline__ int find(const int* start, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Exclusive sum over the CTA's threads in order.  scratch: kThreads / 32 words.
template <int kThreads>
__device__ __forceinline__ long long scan(long long v, long long* scratch, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(FULL_MASK, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();  // scratch may still be read from an earlier scan
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; w++) {
        const long long s = scratch[w];
        if (w < warp) before += s;
        all += s;
    }
    *total = all;
    return before + inc - v;
}

// All threads of the CTA call it.  starts: n_seq + 1 ints of shared memory that stay (the
// first tile of each sequence); share: one Share in shared memory, valid after the call.
template <int kThreads, int kRows, int kBlock, int kMinUnits>
__device__ void find_share(const PagedAttnArgs& a, int* starts, Share* share) {
    __shared__ long long scratch[kThreads / 32];
    const int tid = threadIdx.x, n = a.n_seq;
    const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    int mine = 0;
    for (int i = i0; i < i1; i++) {
        const int tiles = (load_seq(a, i).count * a.group + kRows - 1) / kRows;
        starts[i] = tiles;
        mine += tiles;
    }
    long long all_tiles;
    int at = (int)scan<kThreads>(mine, scratch, &all_tiles);  // (the host bounds rows * group to 31 bits)
    const int n_tiles = (int)all_tiles;
    for (int i = i0; i < i1; i++) {
        const int tiles = starts[i];
        starts[i] = at;
        at += tiles;
    }
    if (tid == 0) starts[n] = n_tiles;
    __syncthreads();
    // units of this thread's run of tiles
    const int pt = (n_tiles + kThreads - 1) / kThreads, g0 = min(n_tiles, tid * pt), g1 = min(n_tiles, g0 + pt);
    long long units = 0;
    if (g0 < g1) {
        int i = find(starts, n, g0);
        Seq s = load_seq(a, i);
        for (int g = g0; g < g1; g++) {
            while (starts[i + 1] <= g) s = load_seq(a, ++i);
            Tile t;
            tile_range<kRows, kBlock>(a, s, (g - starts[i]) * kRows, t);
            units += t.nb;
        }
    }
    long long per_head;
    const long long before = scan<kThreads>(units, scratch, &per_head);
    const long long total = per_head * a.n_kv;
    const int ctas = (int)min((long long)gridDim.x, (total + kMinUnits - 1) / kMinUnits);
    const int c = blockIdx.x;
    if (c >= ctas) {
        if (tid == 0) {
            share->left = 0;
            share->ctas = ctas;
        }
    } else {
        const long long u0 = total * c / ctas, u1 = total * (c + 1) / ctas;
        const int kvh = (int)(u0 / per_head);
        long long x = u0 - kvh * per_head;
        if (x >= before && x < before + units) {  // one thread: its run holds the first unit
            int i = find(starts, n, g0), g = g0;
            Seq s = load_seq(a, i);
            x -= before;
            for (;;) {
                while (starts[i + 1] <= g) s = load_seq(a, ++i);
                Tile t;
                tile_range<kRows, kBlock>(a, s, (g - starts[i]) * kRows, t);
                if (x < t.nb) break;
                x -= t.nb;
                g++;
            }
            share->tile = g;
            share->kvh = kvh;
            share->skip = (int)x;
            share->left = u1 - u0;
            share->n_tiles = n_tiles;
            share->ctas = ctas;
            share->units = total;
        }
    }
    __syncthreads();
}

// Goes through a share segment by segment: blocks [first, first + n) of tile t.
template <int kRows, int kBlock>
struct Walk {
    Share sh;
    const int* starts;
    int seq_hint = 0;
    Tile t;
    int first, n;     // blocks of this segment
    bool head, whole; // the segment begins its tile; it is the whole tile

    __device__ __forceinline__ Walk(const Share& s, const int* st) : sh(s), starts(st) {}
    __device__ __forceinline__ bool next(const PagedAttnArgs& a) {
        if (sh.left <= 0) return false;
        if (sh.tile == sh.n_tiles) {
            sh.tile = 0;
            sh.kvh++;
        }
        const int i = starts[seq_hint] <= sh.tile && sh.tile < starts[seq_hint + 1] ? seq_hint
                                                                                  : find(starts, a.n_seq, sh.tile);
        seq_hint = i;
        t.seq = i;
        t.kvh = sh.kvh;
        tile_range<kRows, kBlock>(a, load_seq(a, i), (sh.tile - starts[i]) * kRows, t);
        first = t.b0 + sh.skip;
        head = sh.skip == 0;
        n = (int)min((long long)(t.nb - sh.skip), sh.left);
        whole = head && n == t.nb;
        sh.left -= n;
        sh.skip = 0;
        sh.tile++;
        return true;
    }
    // The CTAs that share the tile of the present segment (a segment that is not the whole tile).
    __device__ __forceinline__ void sharers(int* c0, int* c1) const {
        const long long share0 = sh.units * blockIdx.x / sh.ctas, share1 = sh.units * (blockIdx.x + 1) / sh.ctas;
        // a segment that does not begin its tile is the share's first; one that does, but does not end it, its last
        const long long u0 = head ? share1 - n : share0 - (first - t.b0), u1 = u0 + t.nb - 1;
        *c0 = (int)(((u0 + 1) * sh.ctas - 1) / sh.units);
        *c1 = (int)(((u1 + 1) * sh.ctas - 1) / sh.units);
    }
};

// Leaves the tile of the present segment, which this CTA begins and others end, to paged_join_kernel.
template <typename W>
__device__ __forceinline__ void join_later(const PagedAttnArgs& a, const W& w) {
    int c0, c1;
    w.sharers(&c0, &c1);
    a.join[blockIdx.x] = PagedJoin{c1, w.t.r0, w.t.rows, w.t.s.row0, w.t.kvh};
}

}  // namespace paged
}  // namespace rbt
