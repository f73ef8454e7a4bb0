// paged_tc.cu -- attention over a paged KV cache for chunks of new tokens, bf16, on the
// 5th-generation tensor cores (tcgen05, TMEM, TMA).
//
// One CTA per SM takes an equal share of the units (paged_sched.cuh); a unit is 256
// query rows (two M = 128 tiles) against 128 positions.  S_i = Q_i K^T goes to TMEM, a
// warpgroup per tile (thread = row) takes the softmax of its row and writes the weights
// P_i, rounded to bf16, over S_i in TMEM, and O_i += P_i V reads P_i from there, so the
// weights never pass through shared memory.  The two tiles alternate: while one has its
// exponentials computed, the other has its products.  TMEM: S_0 S_1 O_0 O_1, all 512
// columns.
//
// A row's maximum m moves only when a block's exceeds it by more than 2^8 in the
// weights; then the row's O in TMEM is rescaled (rare: the maximum settles early), and
// the weights stay below 2^8.  v is the B operand as it lies in the pages (positions x
// dims, "MN-major"), k likewise K-major: no transposed copy of the cache is made.
//
// Warps 0-3 and 4-7: the softmax of tiles 0 and 1; warp 8 issues the MMAs; warp 9 the
// copies.  Every wait is bounded; one that runs out leaves a code, and every role goes on
// without waiting, so that the CTA ends.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/rbt_moe.h"
#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "paged_sched.cuh"
#include "tc_ptx.cuh"

namespace rbt {
namespace {

using namespace paged;
using namespace tc;

constexpr int kTcTile = 128;               // rows of one MMA tile
constexpr int kTcRows = kPagedTcRows;      // two tiles
constexpr int kTcBlock = 128;              // positions of a block
constexpr int kTcThreads = 320;
constexpr uint64_t kTcWaitNs = 2000000000ull;
constexpr float kTcRescale = 8.0f;         // log2 of the largest weight before the maximum moves

template <int HD>
struct TcCfg {
    static constexpr int kStages = HD == 128 ? 2 : 4;
    static constexpr int kHalf = 128 * 128;                 // 128 rows of 64 dims, 128-byte swizzle
    static constexpr int kTileBytes = (HD / 64) * kHalf;    // Q tile, k block or v block
    static constexpr int oQ = 0;
    static constexpr int oK = 2 * kTileBytes;
    static constexpr int oV = oK + kStages * kTileBytes;
    static constexpr int oEnd = oV + kStages * kTileBytes;
    static constexpr int kSmem = oEnd + 1024;
    static constexpr int cS = 0, cO = 256;                  // TMEM columns: S_i at cS + 128 i, O_i at cO + 128 i
};

struct TcBars {
    uint64_t q_full[2], s_full[2], p_full[2], pv_done[2];
    uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
    uint64_t drain;
    uint32_t tmem;
};

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem desc], bf16 A packed two per column
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}

// Descriptor of v as an MN-major B operand in the 128-byte swizzle: rows (positions, the K
// side) of 64 dims; groups of 8 positions 1024 bytes apart, 64-dim halves `half` bytes apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t smem_addr, uint32_t half) {
    const uint64_t lo = (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)((half >> 4) & 0x3FFFu) << 16);
    const uint64_t hi = (uint64_t)(1024u >> 4) | (1ull << 14) | (2ull << 29);
    return lo | (hi << 32);
}

__device__ __forceinline__ uint32_t sw128(int r, int c) {  // 16-byte chunk c of 128-byte row r
    return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}

// A wait that gives up once, for good: the softmax then passes its other barriers at once.
struct Waiter {
    bool ok = true;
    unsigned* status;
    __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait_bounded(bar, parity, kTcWaitNs)) {
            ok = false;
            atomicCAS(status, 0u, (unsigned)kPagedWait);
        }
    }
    // for a whole warp, which goes on only if every lane may
    __device__ __forceinline__ bool warp(uint64_t* bar, uint32_t parity) {
        (*this)(bar, parity);
        return ok = __all_sync(FULL_MASK, ok);
    }
};

template <int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const PagedAttnArgs a) {
    using C = TcCfg<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int* starts = reinterpret_cast<int*>(smem + C::oEnd);
    __shared__ TcBars bars;
    __shared__ Share share;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.q_full[i], kTcTile);
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_full[i], kTcTile);
            mbar_init(&bars.pv_done[i], 1);
        }
        for (int i = 0; i < C::kStages; i++) {
            mbar_init(&bars.k_full[i], 1);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_full[i], 1);
            mbar_init(&bars.v_empty[i], 1);
        }
        mbar_init(&bars.drain, 1);
        fence_mbar_init();
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        a.join[blockIdx.x].last = blockIdx.x;
    }
    if (warp == 8) {
        tmem_alloc(&bars.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    find_share<kTcThreads, kTcRows, kTcBlock, 1>(a, starts, &share);
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    Walk<kTcRows, kTcBlock> w(share, starts);
    Waiter wait;
    wait.status = a.status;

    if (warp == 9) {
        // ------------------------------------------------ copies
        const int box = min(1 << a.page_shift, kTcBlock), n_box = kTcBlock / box, box_shift = min(a.page_shift, 7);
        uint32_t j = 0;
        while (w.next(a)) {
            const int32_t* table = a.table + (size_t)w.t.seq * a.table_stride;
            for (int b = w.first; b < w.first + w.n; b++, j++) {
                const uint32_t st = j % C::kStages, par = (j / C::kStages - 1) & 1;
                const int p0 = b * kTcBlock, left = min(kTcBlock, w.t.hi - p0);
                const int boxes = left > 0 ? (left + box - 1) / box : 0;
                // lane: box lane % n_box of half lane / n_box, .. (at most 16 boxes x 2 halves)
                const int mine = lane & (n_box - 1), half = lane >> (7 - box_shift);
                const bool on = mine < boxes && half < HD / 64;
                int y = 0;
                if (on) {
                    const int p = p0 + mine * box;
                    int id = table[p >> a.page_shift];
                    if ((unsigned)id >= (unsigned)a.n_pages) {  // no page: any valid memory, and no result
                        atomicCAS(a.status, 0u, (unsigned)kPagedTable);
                        id = 0;
                    }
                    y = ((id * a.n_kv + w.t.kvh) << a.page_shift) + (p & ((1 << a.page_shift) - 1));
                }
                const uint32_t bytes = boxes * box * HD * 2;
                const uint32_t at = half * C::kHalf + mine * box * 128;
                if (j >= C::kStages && !wait.warp(&bars.k_empty[st], par)) break;
                if (lane == 0) mbar_arrive_expect_tx(&bars.k_full[st], bytes);
                __syncwarp();
                if (on) tma_load_3d(smem + C::oK + st * C::kTileBytes + at, &tm_k, &bars.k_full[st], 0, y, half);
                if (j >= C::kStages && !wait.warp(&bars.v_empty[st], par)) {  // (k's copies of this block are in flight)
                    wait.ok = true;
                    wait(&bars.k_full[st], (j / C::kStages) & 1);
                    wait.ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(&bars.v_full[st], bytes);
                __syncwarp();
                if (on) tma_load_3d(smem + C::oV + st * C::kTileBytes + at, &tm_v, &bars.v_full[st], 0, y, half);
            }
            if (!wait.ok) break;
        }
        // every copy has landed before the CTA may exit
        wait.ok = true;
        for (uint32_t i = j > C::kStages ? j - C::kStages : 0; i < j; i++) {
            wait(&bars.k_full[i % C::kStages], (i / C::kStages) & 1);
            wait(&bars.v_full[i % C::kStages], (i / C::kStages) & 1);
        }
    } else if (warp == 8) {
        // ------------------------------------------------ MMAs (lane 0 issues)
        constexpr uint32_t idS = idesc_bf16_f32(kTcTile, kTcBlock);
        constexpr uint32_t idO = idesc_bf16_f32(kTcTile, HD) | (1u << 16);  // B is MN-major
        uint32_t j0 = 0, nq[2] = {0, 0}, np[2] = {0, 0};  // blocks before this segment; phases used of q_full, and p_full
        const auto issue_s = [&](int i, uint32_t st) {
            if (lane == 0) {
                const uint32_t sq = smem_u32(smem + C::oQ + i * C::kTileBytes);
                const uint32_t sk = smem_u32(smem + C::oK + st * C::kTileBytes);
#pragma unroll
                for (int kk = 0; kk < HD / 16; kk++) {
                    const uint32_t o = (kk >> 2) * C::kHalf + (kk & 3) * 32;
                    mma_bf16(tmem + C::cS + i * 128, sw128_kmajor_desc(sq + o), sw128_kmajor_desc(sk + o), idS, kk != 0);
                }
                mma_commit(&bars.s_full[i]);
            }
            __syncwarp();
        };
        const auto segment = [&]() -> bool {
            const int nt = w.t.rows > kTcTile ? 2 : 1;
            for (int i = 0; i < nt; i++) {
                if (!wait.warp(&bars.q_full[i], nq[i] & 1)) return false;
                nq[i]++;
                if (i == 0 && !wait.warp(&bars.k_full[j0 % C::kStages], (j0 / C::kStages) & 1)) return false;
                tc_fence_after();
                issue_s(i, j0 % C::kStages);  // (S_i is free: the product that read P_i was waited for)
            }
            if (lane == 0) mma_commit(&bars.k_empty[j0 % C::kStages]);
            for (int n = 0; n < w.n; n++) {
                const uint32_t j = j0 + n, st = j % C::kStages, st1 = (j + 1) % C::kStages;
                for (int i = 0; i < nt; i++) {
                    if (i == 0) {
                        if (!wait.warp(&bars.v_full[st], (j / C::kStages) & 1)) return false;
                        const int p0 = (w.first + n) * kTcBlock;
                        if (p0 + kTcBlock > w.t.hi) {
                            // what lies behind the last position is not a number, perhaps, which a weight of 0 would not hide
                            const int r0 = max(0, w.t.hi - p0);
                            for (int e = lane; e < (kTcBlock - r0) * (HD / 8); e += 32) {
                                const int r = r0 + e / (HD / 8), c = e % (HD / 8);
                                *reinterpret_cast<uint4*>(smem + C::oV + st * C::kTileBytes + (c >> 3) * C::kHalf +
                                                          sw128(r, c & 7)) = make_uint4(0, 0, 0, 0);
                            }
                            fence_async_smem();
                            __syncwarp();
                        }
                    }
                    if (!wait.warp(&bars.p_full[i], np[i] & 1)) return false;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t sv = smem_u32(smem + C::oV + st * C::kTileBytes);
#pragma unroll
                        for (int kk = 0; kk < kTcBlock / 16; kk++)
                            mma_bf16_ts(tmem + C::cO + i * 128, tmem + C::cS + i * 128 + kk * 8, mn_desc(sv + kk * 2048, C::kHalf),
                                        idO, (n | kk) != 0);
                        mma_commit(&bars.pv_done[i]);
                        if (i == nt - 1) mma_commit(&bars.v_empty[st]);
                    }
                    __syncwarp();
                    // S_i of the next block takes the place of P_i: after the product that reads P_i, which the
                    // softmax also counts on (O_i is at rest whenever s_full[i] arrives)
                    if (!wait.warp(&bars.pv_done[i], np[i] & 1)) return false;
                    np[i]++;
                    if (n + 1 < w.n) {
                        if (i == 0 && !wait.warp(&bars.k_full[st1], ((j + 1) / C::kStages) & 1)) return false;
                        tc_fence_after();
                        issue_s(i, st1);
                        if (i == nt - 1 && lane == 0) mma_commit(&bars.k_empty[st1]);
                    }
                }
            }
            j0 += w.n;
            return true;
        };
        while (w.next(a))
            if (!segment()) break;
        // every MMA has completed before TMEM is freed
        if (lane == 0) mma_commit(&bars.drain);
        __syncwarp();
        wait.ok = true;
        wait(&bars.drain, 0);
        __syncwarp();
    } else {
        // ------------------------------------------------ softmax: thread = row
        const int i = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lanes + C::cS + i * 128, tO = tmem + lanes + C::cO + i * 128;
        // a negative scale turns the sign of q instead; a scale of 0 stays above it, so that -inf stays -inf
        const float k2 = fmaxf(fabsf(a.scale) * kLog2e, 1e-37f);
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        uint32_t ns = 0;  // phases used of s_full and pv_done
        while (w.next(a)) {
            const Tile& t = w.t;
            const int row = i * kTcTile + r;  // in the unit
            if (t.rows <= i * kTcTile) continue;
            const bool live = row < t.rows;
            const int tok = (t.r0 + row) / a.group, head = t.kvh * a.group + (t.r0 + row) - tok * a.group;
            const int pos = t.off + tok;
            const int to = !live ? 0 : a.causal ? min(t.s.len, pos + 1) : t.s.len;
            const int from = a.window ? max(0, pos - a.window + 1) : 0;
            {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                                  (t.s.row0 + tok) * a.q_stride + (size_t)head * HD);
                uint8_t* dst = smem + C::oQ + i * C::kTileBytes;
#pragma unroll
                for (int c = 0; c < HD / 8; c++) {
                    uint4 x = live ? src[c] : make_uint4(0, 0, 0, 0);
                    x.x ^= flip;
                    x.y ^= flip;
                    x.z ^= flip;
                    x.w ^= flip;
                    *reinterpret_cast<uint4*>(dst + (c >> 3) * C::kHalf + sw128(r, c & 7)) = x;
                }
                fence_async_smem();
                tc_fence_before();
                mbar_arrive(&bars.q_full[i]);
            }
            float m = -INFINITY, l = 0.0f;
            for (int n = 0; n < w.n; n++) {
                const int p0 = (w.first + n) * kTcBlock;
                wait(&bars.s_full[i], ns & 1);
                ns++;
                __syncwarp();
                tc_fence_after();
                uint32_t v[128];
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[32 * c]));
                tmem_ld_wait();
                float top = -INFINITY;
                const int c0 = from - p0, c1 = to - p0;  // columns [c0, c1) are seen
                if (__all_sync(FULL_MASK, c0 <= 0 && c1 >= kTcBlock)) {
#pragma unroll
                    for (int c = 0; c < 128; c++) top = fmaxf(top, __uint_as_float(v[c]));
                } else {
#pragma unroll
                    for (int c = 0; c < 128; c++) {
                        if (c < c0 || c >= c1) v[c] = 0xff800000u;
                        top = fmaxf(top, __uint_as_float(v[c]));
                    }
                }
                // (equal infinities need no step; m = -inf until the row sees something)
                const bool move = top > m && (m == -INFINITY || (top - m) * k2 > kTcRescale);
                float alpha = 1.0f;
                if (move) {
                    alpha = m == -INFINITY ? 0.0f : ex2((m - top) * k2);
                    m = top;
                    l *= alpha;
                }
                if (n > 0 && __any_sync(FULL_MASK, move)) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(tO + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st_32x32b_x32(tO + c, o);
                    }
                }
                const float mk = m == -INFINITY ? 0.0f : m * k2;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t p[32];
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < 32; c++) {
                        const float x = ex2(fmaf(__uint_as_float(v[64 * h + 2 * c]), k2, -mk));
                        const float y = ex2(fmaf(__uint_as_float(v[64 * h + 2 * c + 1]), k2, -mk));
                        sum[c & 3] += x + y;
                        const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
                        p[c] = *reinterpret_cast<const uint32_t*>(&b);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_st_32x32b_x32(tS + 32 * h, p);
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bars.p_full[i]);
            }
            wait(&bars.pv_done[i], (ns - 1) & 1);
            __syncwarp();
            tc_fence_after();
            const float scale = w.whole ? (l > 0.0f || l != l ? 1.0f / l : 0.0f) : 1.0f;
            const float ml = m == -INFINITY ? -INFINITY : m * k2;
            float* part = a.part + ((size_t)blockIdx.x * 2 + (w.head ? 1 : 0)) * paged_part_floats(kTcRows, HD);
            if (live) {
                if (!w.whole) {
                    part[row] = ml;
                    part[kTcRows + row] = l;
                } else if (a.lse) {
                    a.lse[(size_t)(t.s.row0 + tok) * a.n_heads + head] = l == 0.0f ? -INFINITY : ml * kLn2 + logf(l);
                }
            }
            uint16_t* out = static_cast<uint16_t*>(a.out) + (t.s.row0 + tok) * a.out_stride + (size_t)head * HD;
            float* po = part + paged_part_o(kTcRows) + (size_t)row * HD;
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(tO + c, o);
                tmem_ld_wait();
                if (!live) continue;
                if (w.whole) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t b[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const __nv_bfloat162 x = __floats2bfloat162_rn(__uint_as_float(o[e + 2 * k]) * scale,
                                                                           __uint_as_float(o[e + 2 * k + 1]) * scale);
                            b[k] = *reinterpret_cast<const uint32_t*>(&x);
                        }
                        *reinterpret_cast<uint4*>(out + c + e) = make_uint4(b[0], b[1], b[2], b[3]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(po + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            tc_fence_before();
            if (!w.whole && w.head && threadIdx.x == 0)
                a.join[blockIdx.x] = PagedJoin{w.finisher(), t.r0, t.rows, t.s.row0, t.kvh};
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int HD>
cudaError_t tc_case(const PagedMaps& maps, const PagedAttnArgs& a, int ctas, cudaStream_t s) {
    using C = TcCfg<HD>;
    static_assert(C::kSmem + (kPagedMaxSeq + 1) * 4 + 1024 <= 232448, "shared memory per CTA");
    cudaError_t e = cudaFuncSetAttribute(paged_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         C::kSmem + (kPagedMaxSeq + 1) * 4);
    if (e != cudaSuccess) return e;
    paged_tc_kernel<HD><<<ctas, kTcThreads, C::kSmem + (a.n_seq + 1) * 4, s>>>(maps.k_tc, maps.v_tc, a);
    return cudaGetLastError();
}

}  // namespace

bool paged_tc_maps(PagedMaps* maps, const void* k, const void* v, int hd, int page_size, uint64_t rows) {
    const uint64_t dims[3] = {64, rows, (uint64_t)hd / 64}, strides[2] = {(uint64_t)hd * 2, 128};
    const uint32_t box[3] = {64, (uint32_t)(page_size < kTcBlock ? page_size : kTcBlock), 1};
    return make_map_sw128(&maps->k_tc, k, 3, dims, strides, box) && make_map_sw128(&maps->v_tc, v, 3, dims, strides, box);
}

cudaError_t launch_paged_tc(int hd, const PagedMaps& maps, const PagedAttnArgs& a, int ctas, cudaStream_t s) {
    return hd == 64 ? tc_case<64>(maps, a, ctas, s) : tc_case<128>(maps, a, ctas, s);
}

}  // namespace rbt
