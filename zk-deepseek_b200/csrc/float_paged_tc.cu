// Attention of new tokens over pages on the tensor cores, bfloat16 operands, 32-bit scores, weights and sums.  How the work is
// shared, and what becomes of an item that several CTAs take parts of, is in float_paged.cuh.
//
// paged_stream_kernel: up to 16 query rows (tokens of the step times heads of a group) per key head, so that keys and values are read once
// and their bytes are the bound.  A warp works by itself: it owns every fourth stretch of 16 keys, loads it by TMA into a ring of its
// own and keeps maxima, sums and the weighted values of all 16 rows in registers (m16n8k16 products: queries are the
// A operand and stay in registers, keys and values are read from the swizzled tiles by ldmatrix).  No warp waits for
// another one before the item ends.  Calls among others, the merge of cut items included: 64 sequences up to 8192, 16 key heads of 128, 88 us,
// 5.4 TB/s; one sequence of 4095, 8 key heads, 13.2.
//
// paged_tile_kernel: more rows.  An item is two tiles of up to 128 rows over tiles of 128 keys: scores and outputs of both in tensor
// memory, bfloat16 weights overwrite their scores and are the tensor-memory operand of the second product; while one tile is
// in its softmax the tensor core works for the other.  The rows of a tile are (token, head) pairs, so that all heads of a
// group share the keys that they read.
//   warp 0      the parts of items that the CTA takes, TMA loads
//   warp 1      MMA issue
//   warps 2-9   softmax, tile 0    warps 10-17 softmax, tile 1: two threads share a query row, half of the columns each
// The running maximum only replaces the one in use when it has grown by more than 2^8, and then in front of the next tile, where the
// output tile is rescaled in place: a tile's weights are made from the maximum in use, without looking for the new one first.  A row whose
// scores outgrow that by more than 2^100 within one tile is marked by a sum that is NaN, and is taken again.  Values behind the end of the
// sequence are blanked: what another owner left there would make rows not finite.  Weights go to the second product in halves, so that it
// starts under the other half.  CTAs stay and take one part of an item after the other.  What bounds it is one tile's softmax under the other's
// products: a call for a prompt of 4096, 32 heads of 128 over 8, takes 182 us among others, 0.76 PFLOP/s, the tensor pipe active for 44 %, the
// exponentials' for as much.
#include <cuda.h>

#include "float_paged.cuh"
#include "tcgen05.cuh"

namespace zkds {

bool fp_tensor_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes,
                   const uint32_t* box);

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// mbar_wait_warp without a time to be parked for, for the warp that the tensor core waits for (a prompt of 4096: 175 -> 170 us)
__device__ __forceinline__ bool wait_awake(uint32_t bar, uint32_t parity, volatile int* abort_flag)
{
    for (uint32_t it = 0; it < kSpinLimit * 4; ++it) {
        if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
        if ((it & 255u) == 255u && __any_sync(0xffffffffu, *abort_flag)) return false;
    }
    *abort_flag = 1;
    return false;
}

// ---- few rows ----------------------------------------------------------------------------------------------------
constexpr int kStreamWarps = 4, kStretch = 16, kStreamRows = 16, kStreamKeys = kStreamWarps * kStretch, kStreamMost = 128;
constexpr int kStretchSeg = kStretch * 128;            // bytes of 16 keys x 64 columns
constexpr int kStreamStages = 4;
// An item by itself costs about as much as 6 blocks of 64 keys, or 2 tiles of 128 (64 sequences up to 8192, microseconds, at 2, 3, 4, 5, 6: 127,
// 110, 95, 91, 88; a chunk beside decoding sequences at 2, 3, 4: 116, 117, 119; a prompt 170, 171, 175; today 84, 103 and 167; launches by themselves).  No CTA takes less than
// 4 blocks, or 2 tiles.
constexpr int kStreamOver = 6, kStreamLeast = 2, kTileOver = 2, kTileLeast = 1;

struct StreamShape {
    int segk, segv, box, stages;
    size_t smem;
    StreamShape(const zkfp_paged_attention_args& a)
    {
        segk = (a.d + 63) / 64;
        segv = (a.dv + 63) / 64;
        box = a.page < kStretch ? a.page : kStretch;
        const size_t fixed = 1024 + plan_bytes(a.batch) + kStreamWarps * (kStreamStages * 8 + 2 * kStreamRows * 4 + 8) + 16;
        const size_t load = (size_t)(segk + segv) * kStretchSeg, least = (size_t)segv * 4096;
        const size_t stage = kStreamWarps * (load > least ? load : least), room = 112 * 1024 - fixed;
        stages = (int)(room / stage < kStreamStages ? room / stage : kStreamStages);
        smem = fixed + stages * stage;
    }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Where a warp stands: the part of an item that the CTA takes, and the block of keys that comes next.
struct Cursor {
    Walk w;
    long long u, item_end;           // behind this part; behind the item
    int j, j_end, lo, hi;            // blocks of the part; the positions that any row of the item sees
    bool begins, whole;

    // the part that starts at u, or the next one that has blocks
    __device__ __forceinline__ bool part(const Paged& p, const Plan& plan, long long u1)
    {
        for (;;) {
            const int left = w.left(p), taken = (int)min((long long)left, u1 - u);
            j = w.begin(p);
            j_end = w.end(p, taken);
            item_end = u + left;
            u += taken;
            if (j < j_end) break;
            if (u >= u1) return false;
            w.next(p, plan);
        }
        begins = j == 0;
        whole = begins && j_end == w.count;
        const int base = w.len - w.n, last_row = min((w.t + 1) * p.tile, w.n * p.group) - 1;
        hi = base + by_group(p, last_row);
        lo = first_seen(p, base + by_group(p, w.t * p.tile));
        return true;
    }
    __device__ __forceinline__ bool next(const Paged& p, const Plan& plan, long long u1)
    {
        if (u >= u1) return false;
        w.next(p, plan);
        return part(p, plan, u1);
    }
};

template <int SEGK, int SEGV>
__global__ void __launch_bounds__(kStreamWarps * 32, 2)
paged_stream_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ Paged p, int box, int stages)
{
    extern __shared__ uint8_t raw[];
    const zkfp_paged_attention_args& a = p.a;
    constexpr uint32_t kLoad = (SEGK + SEGV) * kStretchSeg, kStage = kLoad > SEGV * 4096 ? kLoad : SEGV * 4096;      // also room for 16 rows of sums
    constexpr int kPitch = SEGV * 64;
    uint8_t* ring = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, batch = (int)a.batch, dv = a.dv;
    uint64_t* bars = (uint64_t*)(ring + kStreamWarps * stages * kStage);           // [warp][stage]
    float* M = (float*)(bars + kStreamWarps * kStreamStages);                      // [warp][row], and the sums of weights
    float* L = M + kStreamWarps * kStreamRows;
    const uint8_t** sums = (const uint8_t**)(L + kStreamWarps * kStreamRows);      // where a warp left its rows
    int* gave_up = (int*)(sums + kStreamWarps);
    const Plan plan((uint8_t*)(gave_up + 4), batch);
    volatile int* abort_flag = gave_up;
    if (threadIdx.x == 0) {
        *gave_up = 0;
        for (int i = 0; i < kStreamWarps * stages; ++i) mbar_init(smem_u32(bars + i), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_enter();                                     // barriers touch nobody else
    if (threadIdx.x == 0) no_cut(p, blockIdx.x);
    make_plan(p, plan);
    const long long units = plan.before[batch];
    const Share share(p, units);
    const int cta = blockIdx.x;
    if (cta >= share.ctas || units == 0) return;
    const long long u1 = share.begin(cta + 1);
    const uint32_t one = elect_one(), my_bars = smem_u32(bars + warp * stages);
    uint8_t* my_ring = ring + warp * stages * kStage;
    Cursor at;
    at.u = share.begin(cta);
    at.w.locate(p, plan, at.u);
    bool more = at.part(p, plan, u1), loads = more, ok = true;
    Cursor in = at;                                            // the loads, as far ahead as the ring holds
    int slot_in = 0, slot = 0, ahead = 0;
    uint32_t phase = 0;
    // pages of the next 32 stretches of the item that is being loaded: lane i holds that of block base + i
    int page_base = -1, page_id = 0, page_id2 = 0;
    auto fill = [&] {
        while (loads && ahead < stages) {
            if (in.j == in.j_end) {
                loads = in.next(p, plan, u1);
                page_base = -1;
                continue;
            }
            const int k0 = (in.w.first + in.j) * kStreamKeys + warp * kStretch;
            if (k0 > in.hi || k0 + kStretch <= in.lo) {        // a stretch that no row sees takes no place
                ++in.j;
                continue;
            }
            if (page_base < 0 || in.j >= page_base + 32) {
                page_base = in.j;
                const int j = in.j + lane;
                page_id = page_id2 = (int)a.pages;             // beyond the tensor: the tile is filled with zeros
                if (j < in.j_end) {
                    const int k = (in.w.first + j) * kStreamKeys + warp * kStretch;
                    bool bad = false;
                    if (k < in.w.len) {
                        const long long page = page_of(p, in.w.b, k);
                        if (page >= 0) page_id = (int)page;
                        else bad = true;
                    }
                    if (box < kStretch && k + 8 < in.w.len) {
                        const long long page = page_of(p, in.w.b, k + 8);
                        if (page >= 0) page_id2 = (int)page;
                        else bad = true;
                    }
                    if (bad) *(volatile int*)(p.error_flag + 1) = 1;
                }
                __syncwarp();
            }
            const int page = __shfl_sync(0xffffffffu, page_id, in.j - page_base), page2 = __shfl_sync(0xffffffffu, page_id2, in.j - page_base);
            const uint32_t bar = my_bars + slot_in * 8, dst = smem_u32(my_ring) + slot_in * kStage;
            const int line = k0 & (a.page - 1);
            mbar_expect_tx(bar, kLoad, one);
#pragma unroll
            for (int c = 0; c < SEGK + SEGV; ++c) {
                const CUtensorMap* map = c < SEGK ? &tmK : &tmV;
                const int x = (c < SEGK ? c : c - SEGK) * 64;
                tma_load_4d(dst + c * kStretchSeg, map, x, in.w.kv, line, page, bar, one);
                if (box < kStretch) tma_load_4d(dst + c * kStretchSeg + 1024, map, x, in.w.kv, 0, page2, bar, one);
            }
            if (++slot_in == stages) slot_in = 0;
            ++ahead;
            ++in.j;
        }
    };
    fill();
    const int r = lane >> 2, cq = (lane & 3) * 2;
    const float scale = a.scale * kLog2e;
    for (; more; more = at.next(p, plan, u1)) {
        const Walk& w = at.w;
        const int row0 = w.t * p.tile, rows = min(p.tile, w.n * p.group - row0), halves = rows > 8 ? 2 : 1;
        if (threadIdx.x == 0 && at.begins && !at.whole) write_cut(p, cta, share, w, at.item_end);
        // queries: rows r and r + 8, elements cq, cq + 1 and eight further on of every 16
        uint32_t q[SEGK * 4][4];
        int pos[2] = {-1, -1};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int k = 0; k < SEGK * 4; ++k) q[k][h] = q[k][h + 2] = 0u;
            if (h >= halves) break;
            const int rr = row0 + r + 8 * h, t = by_group(p, rr), head = w.kv * p.group + rr - t * p.group;
            if (r + 8 * h >= rows) continue;
            pos[h] = w.len - w.n + t;
            const bf16* src = (const bf16*)a.q + (long long)(w.row0 + t) * a.q_tok + head * a.q_head + cq;
#pragma unroll
            for (int k = 0; k < SEGK * 4; ++k) {
                if (k * 16 < a.d) q[k][h] = *(const uint32_t*)(src + k * 16);
                if (k * 16 + 8 < a.d) q[k][h + 2] = *(const uint32_t*)(src + k * 16 + 8);
            }
        }
        const int low_pos = w.len - w.n + by_group(p, row0), all_lo = a.window > 0 ? at.hi - a.window : -1;
        float o[SEGV * 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
        uint8_t* mine = nullptr;                               // the place read last
        for (int j = at.j; j < at.j_end; ++j) {
            const int k0 = (w.first + j) * kStreamKeys + warp * kStretch;
            if (k0 > at.hi || k0 + kStretch <= at.lo) continue;
            fill();
            mine = my_ring + slot * kStage;
            const uint32_t tile = smem_u32(mine);
            if (ok) ok = mbar_wait_warp(my_bars + slot * 8, phase, abort_flag);
            float s[2][4] = {};
#pragma unroll
            for (int k = 0; k < SEGK * 2; ++k) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t b[4];
                    const int key = t * 8 + (lane & 7), chunk = k * 4 + (lane >> 3);
                    ldmatrix4(b, tile + (chunk >> 3) * kStretchSeg + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
                    mma16816(s[t], q[2 * k], b[0], b[1]);
                    mma16816(s[t], q[2 * k + 1], b[2], b[3]);
                }
            }
            // s[t][2 h + e]: row r + 8 h, key k0 + 8 t + cq + e
            const bool edge = k0 + kStretch - 1 > low_pos || k0 <= all_lo;         // some row does not see all of them
            float f[2] = {1.f, 1.f};
            uint32_t pa[4] = {};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= halves) break;
                if (edge) {
                    const int lo = a.window > 0 ? pos[h] - a.window : -1;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = k0 + 8 * t + cq + e;
                            if (key > pos[h] || key <= lo) s[t][2 * h + e] = -INFINITY;
                        }
                }
                float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m_new = fmaxf(m[h], top * scale), m_sub = m_new == -INFINITY ? 0.f : m_new;
                f[h] = exp2_approx(m[h] - m_sub);
                m[h] = m_new;
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = exp2_approx(fmaf(s[i >> 1][2 * h + (i & 1)], scale, -m_sub));
                l[h] = fmaf(l[h], f[h], (e[0] + e[1]) + (e[2] + e[3]));
                pa[h] = pack_bf16(e[0], e[1]);
                pa[h + 2] = pack_bf16(e[2], e[3]);
            }
            if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                for (int c = 0; c < SEGV * 8; ++c) {
                    o[c][0] *= f[0]; o[c][1] *= f[0];
                    o[c][2] *= f[1]; o[c][3] *= f[1];
                }
            }
            if (k0 + kStretch > w.len) {                       // lines that the sequence does not hold: no value, whatever is there
                for (int i = lane; i < SEGV * 128; i += 32)
                    if (k0 + ((i >> 3) & 15) >= w.len) *(uint4*)(mine + (SEGK + (i >> 7)) * kStretchSeg + (i & 127) * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
#pragma unroll
            for (int c = 0; c < SEGV * 4; ++c) {
                uint32_t b[4];
                const int key = (lane & 15), chunk = c * 2 + (lane >> 4);
                ldmatrix4_trans(b, tile + (SEGK + (chunk >> 3)) * kStretchSeg + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
                mma16816(o[2 * c], pa, b[0], b[1]);
                mma16816(o[2 * c + 1], pa, b[2], b[3]);
            }
            __syncwarp();                                      // every lane has read the tile
            --ahead;
            if (++slot == stages) { slot = 0; phase ^= 1u; }
        }
        // The warps' sums meet in the places that they have read last, eight columns at a time turned by the row so that no two rows
        // of a store fall on one bank; a warp that had no keys stays out.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (h >= halves) break;
            if ((lane & 3) == 0) {
                M[warp * kStreamRows + r + 8 * h] = m[h];
                L[warp * kStreamRows + r + 8 * h] = l[h];
            }
            if (mine)
#pragma unroll
                for (int c = 0; c < SEGV * 8; ++c)
                    *(float2*)(mine + ((r + 8 * h) * kPitch + ((c ^ r) * 8) + cq) * 4) = make_float2(o[c][2 * h], o[c][2 * h + 1]);
        }
        if (lane == 0) sums[warp] = mine;
        __syncthreads();
        for (int rr = warp; rr < rows; rr += kStreamWarps) {
            float top = -INFINITY, sum = 0.f, x[1][4] = {};
#pragma unroll
            for (int i = 0; i < kStreamWarps; ++i) top = fmaxf(top, M[i * kStreamRows + rr]);
#pragma unroll
            for (int i = 0; i < kStreamWarps; ++i) {
                const float mi = M[i * kStreamRows + rr];
                if (mi == -INFINITY) {
                    sum += L[i * kStreamRows + rr];            // 0, or NaN where a visible score was
                    continue;
                }
                const float g = exp2_approx(mi - top);
                sum = fmaf(g, L[i * kStreamRows + rr], sum);
                if (lane * 4 < kPitch) {
                    const float4 y = *(const float4*)(sums[i] + (rr * kPitch + (((lane >> 1) ^ (rr & 7)) * 8) + (lane & 1) * 4) * 4);
                    x[0][0] = fmaf(g, y.x, x[0][0]); x[0][1] = fmaf(g, y.y, x[0][1]);
                    x[0][2] = fmaf(g, y.z, x[0][2]); x[0][3] = fmaf(g, y.w, x[0][3]);
                }
            }
            if (at.whole) {
                finish_row<bf16>(p, w, row0 + rr, x, sum);
                continue;
            }
            const long long to = (2ll * cta + (at.begins ? 1 : 0)) * p.tile + rr;
            if (lane * 4 < dv) store4(p.part + to * dv + lane * 4, x[0]);
            if (lane == 0) *(float2*)(p.ml + to * 2) = make_float2(top, sum);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");               // the places are loaded into again
        __syncthreads();
        fill();
    }
    if (!ok) *(volatile int*)p.error_flag = 1;
}

// ---- many rows ---------------------------------------------------------------------------------------------------
constexpr int kTile = 128;                     // query rows and keys per tile
constexpr uint32_t kSeg = kTile * 128;         // bytes of 128 rows x 64 bfloat16
constexpr int kTileThreads = 576, kTileMost = 128;
constexpr int kMaxKeySlots = 8;
// log2 of how far a tile's scores may be above the maximum in use, so that neither its sums (128 weights) nor the factor that brings them down
// in front of the next tile, or where parts are merged, leave the range of 32 bits (factors below 2^-126 are flushed to zero).  Looked at where the
// maximum is replaced and behind the last tile; behind every tile costs a prompt of 4096 3 %.
constexpr float kMostGrown = 100.f;

struct TileParams {
    Paged p;
    int rows;                                  // query rows of a tile: whole groups, up to 128
    int box;                                   // lines of a page in one load
    int seg, segv, k_slots, v_stages;          // segments of 64 columns, ring of key segments, value tiles
    float scale_log2;
};

// The part of an item that a CTA takes: tiles of keys begin .. end - 1 in units of kTile positions (none: no part follows), those that query
// tile g takes part in, and the rows of g.
struct Part {
    int begin, end, row0[2], rows[2], first[2], last[2];
    int b, kv, token0, base, len;              // sequence, key head, first token of the sequence, position of that, positions of the sequence
    int begins, whole;
};

__device__ __forceinline__ Part part_of(const TileParams& t, const Walk& w, int taken)
{
    Part x;
    const int all = w.n * t.p.group;
    x.begin = w.begin(t.p);
    x.end = w.end(t.p, taken);
    x.begins = x.begin == 0;
    x.whole = x.begins && x.end == w.count;
    x.begin += w.first;
    x.end += w.first;
    x.b = w.b;
    x.kv = w.kv;
    x.token0 = w.row0;
    x.base = w.len - w.n;
    x.len = w.len;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        x.row0[g] = w.t * t.p.tile + g * t.rows;
        x.rows[g] = max(0, min(t.rows, all - x.row0[g]));
        const int i0 = x.base + by_group(t.p, x.row0[g]), i1 = x.rows[g] > 0 ? x.base + by_group(t.p, x.row0[g] + x.rows[g] - 1) : -1;
        x.first[g] = max(x.begin, first_seen(t.p, i0) / kTile);
        x.last[g] = i1 >= 0 ? min(x.end - 1, i1 / kTile) : x.first[g] - 1;
    }
    return x;
}

struct TileShared {
    uint64_t q_full, q_empty, k_full[kMaxKeySlots], k_empty[kMaxKeySlots], v_full[2], v_empty[2], s_full[2], p_full[2][2], o_full[2], o_empty[2];
    uint64_t part_full[2], part_empty[2];
    __align__(16) uint8_t stage[16][1024];     // 32 bytes of the 32 rows of a warp
    float most[4][2][2][kTile];                // [use][query tile][half][row], see below
    Part part[2];
    uint32_t tmem;
    int abort;
};

// ---- the scores of a row -----------------------------------------------------------------------------------------
// Two threads share a row, 64 of its scores in tensor memory each: 32 at a time go through registers.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// largest score of 64 columns from c0 on
template <bool MASKED>
__device__ __forceinline__ float tile_max(uint32_t tS, int c0, int c_lo, int c_hi)
{
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        float v[32];
        tmem_ld32(tS + q * 32u, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const int c = c0 + q * 32 + i;
            if (MASKED) {
                if (c < c_lo || c > c_hi) v[i] = -INFINITY;
                if (c + 1 < c_lo || c + 1 > c_hi) v[i + 1] = -INFINITY;
            }
            top[(i >> 1) & 1] = max3(top[(i >> 1) & 1], v[i], v[i + 1]);
        }
    }
    return fmaxf(top[0], top[1]);
}

// bfloat16 weights 2^(score * scale - sub) of the visible ones of 64 columns from c0 on, over their scores.  Gives their sum, and in `top` the
// largest score.
template <bool MASKED>
__device__ __forceinline__ float weigh(uint32_t tS, int c0, int c_lo, int c_hi, uint64_t scale, uint64_t sub, float& top)
{
    float most[2] = {-INFINITY, -INFINITY};
    uint64_t add[2] = {0, 0};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        float v[32];
        uint32_t x[16];
        tmem_ld32(tS + q * 32u, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const int c = c0 + q * 32 + i;
            if (MASKED) {
                if (c < c_lo || c > c_hi) v[i] = -INFINITY;
                if (c + 1 < c_lo || c + 1 > c_hi) v[i + 1] = -INFINITY;
            }
            most[(i >> 1) & 1] = max3(most[(i >> 1) & 1], v[i], v[i + 1]);
            const uint64_t y = fma_pair(pair_of(v[i], v[i + 1]), scale, sub);
            float e, f;
            unpair(y, e, f);
            e = exp2_approx(e);
            f = exp2_approx(f);
            add[(i >> 1) & 1] = add_pair(add[(i >> 1) & 1], pair_of(e, f));
            x[i / 2] = pack_bf16(e, f);
        }
        tmem_st16(tS + q * 16u, x);
    }
    float e, f;
    unpair(add_pair(add[0], add[1]), e, f);
    top = fmaxf(most[0], most[1]);
    return e + f;
}

// Lines of a tile of values from `held` on, which the sequence does not hold: no value, whatever is there.  (A function of its own, out of the way of
// the products: a prompt of 4096 182 us, with it in the loop 185.)
__device__ __noinline__ void blank_lines(uint8_t* tile, int held, int segments)
{
    for (int c = 0; c < segments; ++c)
        for (int i = held * 8 + (threadIdx.x & 31); i < kTile * 8; i += 32) *(uint4*)(tile + (uint32_t)c * kSeg + i * 16) = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

__global__ void __launch_bounds__(kTileThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ TileParams t)
{
    extern __shared__ __align__(1024) uint8_t raw[];
    const Paged& p = t.p;
    const zkfp_paged_attention_args& a = p.a;
    uint8_t* base = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t tile_bytes = (uint32_t)(2 * t.seg + t.k_slots + t.v_stages * t.segv) * kSeg;
    TileShared& s = *reinterpret_cast<TileShared*>(base + tile_bytes);
    const Plan plan(base + tile_bytes + ((sizeof(TileShared) + 15) & ~15), (int)a.batch);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sQ = smem_u32(base), bytesQ = (uint32_t)t.seg * kSeg;
    const uint32_t sK = sQ + 2 * bytesQ, sV = sK + (uint32_t)t.k_slots * kSeg, bytesV = (uint32_t)t.segv * kSeg;
    volatile int* abort_flag = &s.abort;
    if (threadIdx.x == 0) {
        s.abort = 0;
        mbar_init(smem_u32(&s.q_full), 1);
        mbar_init(smem_u32(&s.q_empty), 1);
        for (int i = 0; i < kMaxKeySlots; ++i) {
            mbar_init(smem_u32(&s.k_full[i]), 1);
            mbar_init(smem_u32(&s.k_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s.v_full[i]), 1);
            mbar_init(smem_u32(&s.v_empty[i]), 1);
            mbar_init(smem_u32(&s.s_full[i]), 1);
            mbar_init(smem_u32(&s.p_full[i][0]), 4);
            mbar_init(smem_u32(&s.p_full[i][1]), 4);
            mbar_init(smem_u32(&s.o_full[i]), 1);
            mbar_init(smem_u32(&s.o_empty[i]), 8);
            mbar_init(smem_u32(&s.part_full[i]), 1);
            mbar_init(smem_u32(&s.part_empty[i]), 17);         // the warp of MMAs, sixteen of softmax
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    chain_enter();                                     // barriers touch nobody else
    if (warp == 1) tmem_alloc(smem_u32(&s.tmem), 512);
    make_plan(p, plan);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const long long units = plan.before[a.batch];
    const Share share(p, units);
    const int cta = blockIdx.x;
    const bool works = cta < share.ctas && units > 0;

    if (warp == 0) {
        const uint32_t one = elect_one();
        int ks = 0, vs = 0;
        uint32_t kp = 0, vp = 0, qp = 0;
        bool ok = true;
        long long u = works ? share.begin(cta) : 0;
        const long long u1 = works ? share.begin(cta + 1) : 0;
        Walk w;
        if (works) w.locate(p, plan, u);
        if (one) no_cut(p, cta);
        int slot = 0;
        uint32_t phase = 0;
        Part part;
        auto publish = [&] {
            if (!mbar_wait_warp(smem_u32(&s.part_empty[slot]), phase ^ 1u, abort_flag)) return false;
            if (one) {
                s.part[slot] = part;
                mbar_arrive(smem_u32(&s.part_full[slot]));
            }
            slot ^= 1;
            phase ^= slot == 0 ? 1u : 0u;
            return true;
        };
        while (u < u1 && ok) {
            const int taken = (int)min((long long)w.left(p), u1 - u);
            part = part_of(t, w, taken);
            if (part.begin == part.end) break;                 // units of an item that others take
            if (one && part.begins && !part.whole) write_cut(p, cta, share, w, u + w.left(p));
            if (!(ok = publish())) break;
            if (!(ok = mbar_wait_warp(smem_u32(&s.q_empty), qp ^ 1u, abort_flag))) break;
            qp ^= 1u;
            const uint32_t row_bytes = (uint32_t)t.rows * 128u;
            mbar_expect_tx(smem_u32(&s.q_full), (uint32_t)t.seg * row_bytes * (part.rows[1] > 0 ? 2 : 1), one);
#pragma unroll
            for (int g = 0; g < 2; ++g)
                if (part.rows[g] > 0)
                    for (int c = 0; c < t.seg; ++c)
                        tma_load_4d(sQ + g * bytesQ + c * kSeg, &tmQ, c * 64, 0, w.kv, w.row0 + by_group(p, part.row0[g]), smem_u32(&s.q_full), one);
            for (int j = part.begin; j < part.end && ok; ++j) {
                // pages of this tile of keys: lane i holds that of its i-th box, and asks for it
                int mine = (int)a.pages;                       // beyond the tensor: zeros
                const int at = j * kTile + lane * t.box;
                const uint32_t loads = lane * t.box < kTile;
                if (loads && at < w.len) {
                    const long long page = page_of(p, w.b, at);
                    if (page >= 0) mine = (int)page;
                    else *(volatile int*)(p.error_flag + 1) = 1;
                }
                __syncwarp();
                const int line = (j * kTile) & (a.page - 1);
                for (int c = 0; c < t.seg; ++c) {
                    if (!(ok = mbar_wait_warp(smem_u32(&s.k_empty[ks]), kp ^ 1u, abort_flag))) break;
                    const uint32_t bar = smem_u32(&s.k_full[ks]), dst = sK + (uint32_t)ks * kSeg;
                    mbar_expect_tx(bar, kSeg, one);
                    tma_load_4d(dst + lane * t.box * 128, &tmK, c * 64, w.kv, line, mine, bar, loads);
                    if (++ks == t.k_slots) { ks = 0; kp ^= 1u; }
                }
                if (!ok || !(ok = mbar_wait_warp(smem_u32(&s.v_empty[vs]), vp ^ 1u, abort_flag))) break;
                const uint32_t bar = smem_u32(&s.v_full[vs]), dst = sV + (uint32_t)vs * bytesV;
                mbar_expect_tx(bar, bytesV, one);
                for (int c = 0; c < t.segv; ++c) tma_load_4d(dst + c * kSeg + lane * t.box * 128, &tmV, c * 64, w.kv, line, mine, bar, loads);
                if (++vs == t.v_stages) { vs = 0; vp ^= 1u; }
            }
            u += taken;
            if (u < u1) w.next(p, plan);
        }
        part.begin = part.end = 0;
        if (ok) publish();
    } else if (warp == 1) {
        const uint32_t one = elect_one(), tm = uniform(tmem);
        const uint32_t idesc_s = idesc_bf16(kTile, kTile), idesc_o = idesc_bf16(kTile, (a.dv + 15) & ~15, true);
        uint32_t pp[2] = {0, 0}, op[2] = {0, 0}, kp = 0, vp = 0, qp = 0, phase = 0;
        int ks = 0, vs = 0, at = 0, begin = 0, end = 0, len = 0, first[2] = {0, 0}, last[2] = {0, 0};
        // the sums of query tile g over the keys that are there, and its scores with the tile of keys that follows
        auto values = [&](const int g, int j) {
            if (j == first[g]) {                               // the last part's sums have been read
                if (!wait_awake(smem_u32(&s.o_empty[g]), op[g] ^ 1u, abort_flag)) return false;
                op[g] ^= 1u;
            }
            const uint32_t ta = tm + g * kTile;
            const uint64_t vd = smem_desc_mn_sw128(sV + (uint32_t)vs * bytesV, kSeg);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!wait_awake(smem_u32(&s.p_full[g][h]), pp[g], abort_flag)) return false;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < kTile / 32; ++k)
                    umma_bf16_ts(ta + 256u, ta + (uint32_t)(h * 64 + k * 8), vd + (uint64_t)((h * kTile / 32 + k) * 128), idesc_o, (j != first[g] || h || k) ? 1u : 0u, one);
            }
            pp[g] ^= 1u;
            if (j == last[g]) umma_commit(smem_u32(&s.o_full[g]), one);
            return true;
        };
        // every segment is waited for once (by tile 0) and handed back once (by tile 1), also where neither has a use for it
        auto scores = [&](const int g, int j) {
            const bool use = j >= first[g] && j <= last[g];
            int slot = ks;
            uint32_t ph = kp;
            for (int c = 0; c < t.seg; ++c) {
                if (g == 0) {
                    if (!wait_awake(smem_u32(&s.k_full[slot]), ph, abort_flag)) return false;
                    tc_fence_after();
                }
                if (use) {
                    const int cols = a.d - c * 64;
                    const uint64_t ad = smem_desc_sw128(sQ + g * bytesQ + (uint32_t)c * kSeg), bd = smem_desc_sw128(sK + (uint32_t)slot * kSeg);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k * 16 < cols) umma_bf16(tm + g * kTile, ad + (uint64_t)(k * 2), bd + (uint64_t)(k * 2), idesc_s, (c | k) ? 1u : 0u, one);
                }
                if (g == 1) umma_commit(smem_u32(&s.k_empty[slot]), one);
                if (++slot == t.k_slots) { slot = 0; ph ^= 1u; }
            }
            if (use) umma_commit(smem_u32(&s.s_full[g]), one);
            if (g == 1) { ks = slot; kp = ph; }
            return true;
        };
        for (;;) {
            if (!wait_awake(smem_u32(&s.part_full[at]), phase, abort_flag)) break;
            begin = (int)uniform(s.part[at].begin);
            end = (int)uniform(s.part[at].end);
            len = (int)uniform(s.part[at].len);
            const bool ragged = end > len / kTile;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                first[g] = (int)uniform(s.part[at].first[g]);
                last[g] = __reduce_max_sync(0xffffffffu, s.part[at].last[g]);
            }
            if (one) mbar_arrive(smem_u32(&s.part_empty[at]));
            __syncwarp();
            at ^= 1;
            phase ^= at == 0 ? 1u : 0u;
            if (begin == end || !wait_awake(smem_u32(&s.q_full), qp, abort_flag)) break;
            qp ^= 1u;
            tc_fence_after();
            bool ok = scores(0, begin) && scores(1, begin);
            if (ok && begin + 1 == end) umma_commit(smem_u32(&s.q_empty), one);
            for (int j = begin; j < end && ok; ++j) {
                if (!(ok = wait_awake(smem_u32(&s.v_full[vs]), vp, abort_flag))) break;
                if (ragged && j + 1 == end) blank_lines(base + (sV - sQ) + (uint32_t)vs * bytesV, len & (kTile - 1), t.segv);
                tc_fence_after();
                if (j >= first[0] && j <= last[0]) ok = values(0, j);
                if (ok && j + 1 < end) ok = scores(0, j + 1);
                if (ok && j >= first[1] && j <= last[1]) ok = values(1, j);
                if (!ok) break;
                umma_commit(smem_u32(&s.v_empty[vs]), one);
                if (j + 1 < end) ok = scores(1, j + 1);
                if (j + 2 == end) umma_commit(smem_u32(&s.q_empty), one);
                if (++vs == t.v_stages) { vs = 0; vp ^= 1u; }
            }
            if (!ok) break;
        }
    } else {
        const int g = (warp - 2) >> 3, half = ((warp - 2) >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane, c0 = half * 64;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t tS = tmem + (uint32_t)(g * kTile + c0) + lanes, tO = tmem + 256u + (uint32_t)g * kTile + lanes;
        const int middle = (a.dv / 2 + 15) & ~15, o_begin = half ? middle : 0, o_end = half ? a.dv : min(a.dv, middle);
        const uint64_t scale2 = twice(t.scale_log2);
        auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + quarter) : "memory"); };
        uint32_t sp = 0, op = 0;
        bool ok = true;
        int at = 0;
        uint32_t phase = 0;
        for (;;) {
            if (!(ok = mbar_wait_warp(smem_u32(&s.part_full[at]), phase, abort_flag))) break;
            const Part& part = s.part[at];
            if (part.begin == part.end) break;
            const int rows = part.rows[g], first_tile = part.first[g], last_tile = part.last[g];
            const int in_seq = by_group(p, part.row0[g] + row), pos = row < rows ? part.base + in_seq : -1;
            // the maximum in use (in units of log2), the same in both threads of a row, and this one's sum of weights
            float m = -INFINITY, l = 0.f;
            for (int j = first_tile; j <= last_tile; ++j) {
                if (!(ok = mbar_wait_warp(smem_u32(&s.s_full[g]), sp, abort_flag))) break;
                sp ^= 1u;
                tc_fence_after();
                if (quarter * 32 < rows) {                // a warp without rows leaves the scores as weights that nothing reads
                    // visible columns of this row: c_lo .. c_hi
                    const int c_hi = pos - j * kTile, c_lo = a.window > 0 ? c_hi - a.window + 1 : -1;
                    const bool masked = __any_sync(0xffffffffu, row < rows && (c_hi < kTile - 1 || c_lo > 0));
                    // Both halves' largest scores of the tile in front: a thread leaves its own ahead of its weights, without which the next scores
                    // are not made, in two places by turns.
                    const float top = j == first_tile ? -INFINITY : fmaxf(s.most[j + 1 & 1][g][0][row], s.most[j + 1 & 1][g][1][row]) * t.scale_log2;
                    if (__any_sync(0xffffffffu, top > m + 8.0f && m != -INFINITY)) {
                        const float f = m == -INFINITY ? 1.f : exp2_approx(m - fmaxf(m, top));
                        for (int c = o_begin; c < o_end; c += 8) {
                            int32_t o[8];
                            tmem_ld8(tO + (uint32_t)c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = __float_as_int(__int_as_float(o[i]) * f);
                            tmem_st8(tO + (uint32_t)c, o);
                        }
                        l = top - m > kMostGrown ? __int_as_float(0x7fffffff) : l * f;
                        m = m == -INFINITY ? m : fmaxf(m, top);
                    }
                    if (__any_sync(0xffffffffu, m == -INFINITY)) {      // rows that have not seen a key yet
                        s.most[2][g][half][row] = masked ? tile_max<true>(tS, c0, c_lo, c_hi) : tile_max<false>(tS, c0, 0, 0);
                        pair_sync();
                        if (m == -INFINITY) m = fmaxf(s.most[2][g][0][row], s.most[2][g][1][row]) * t.scale_log2;
                    }
                    const uint64_t sub = twice(m == -INFINITY ? 0.f : -m);
                    float most;
                    if (masked) l += weigh<true>(tS, c0, c_lo, c_hi, scale2, sub, most);
                    else l += weigh<false>(tS, c0, 0, 0, scale2, sub, most);
                    s.most[j & 1][g][half][row] = most;
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s.p_full[g][half]));
            }
            if (!ok) break;
            const bool any = first_tile <= last_tile, writes = quarter * 32 < rows, whole = part.whole;
            const int tok = part.token0 + in_seq, b = part.b, kv = part.kv, head = kv * p.group + part.row0[g] + row - in_seq * p.group;
            const long long slot = (2ll * cta + (part.begins ? 1 : 0)) * p.tile + g * t.rows + row;
            // Of an item that is whole, 32 bytes of every row pass through shared memory, so that a store meets 16 rows and not 32: lanes 2 r and
            // 2 r + 1 take the halves of rows r and r + 16; sums of a part go out 32 bytes a row and store.  Gates come one step ahead, the first under the last products.
            const int piece = lane & 1;
            long long to[2], gate_at[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int who = (lane >> 1) + 16 * k;
                const long long tk = __shfl_sync(0xffffffffu, tok, who), hd = __shfl_sync(0xffffffffu, head, who);
                to[k] = quarter * 32 + who >= rows ? -1 : tk * a.o_tok + hd * a.o_head;
                gate_at[k] = tk * a.gate_tok + hd * a.gate_head;
            }
            const bool gated = whole && a.gate;
            uint4 gate[2];
            auto ask = [&](int col) {
#pragma unroll
                for (int k = 0; k < 2; ++k) gate[k] = gated && to[k] >= 0 && col < o_end ? *(const uint4*)((const bf16*)a.gate + gate_at[k] + col) : make_uint4(0, 0, 0, 0);
            };
            ask(o_begin + 8 * piece);
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s.part_empty[at]));
            at ^= 1;
            phase ^= at == 0 ? 1u : 0u;
            if (any) {
                if (!(ok = mbar_wait_warp(smem_u32(&s.o_full[g]), op, abort_flag))) break;
                op ^= 1u;
                tc_fence_after();
            }
            if (writes) {
                if (any) {                                // (without a tile nothing keeps the halves from the next part's place)
                    if (s.most[last_tile & 1][g][half][row] * t.scale_log2 - m > kMostGrown) l = __int_as_float(0x7fffffff);
                    s.most[3][g][half][row] = l;
                    pair_sync();
                    l += s.most[3][g][half ^ 1][row];
                }
                uint8_t* stage = s.stage[warp - 2];
                auto at_stage = [&](int r, int i) { return (uint4*)(stage + r * 32 + ((i ^ (r >> 2)) & 1) * 16); };
                if (whole) {
                    const uint64_t r2 = twice(pos >= 0 ? 1.0f / l : 0.f);
                    const bool blank = __any_sync(0xffffffffu, pos < 0);
                    __nv_bfloat162 none = __float2bfloat162_rn(0.f);     // stays zero where everything is finite
                    const __nv_bfloat162 zero = none;
#pragma unroll 1
                    for (int c = o_begin; c < o_end; c += 16) {
                        float y[16] = {};
                        if (any) {
                            tmem_ldn(tO + (uint32_t)c, *reinterpret_cast<int32_t(*)[16]>(y));
                            tmem_ld_wait();
                        }
                        const int col = c + 8 * piece;
                        if (a.gate) {
#pragma unroll
                            for (int k = 0; k < 2; ++k) *at_stage((lane >> 1) + 16 * k, piece) = gate[k];
                            ask(col + 16);
                            __syncwarp();
                        }
                        if (blank && pos < 0)
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = 0.f;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t x[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float e, f;
                                unpair(fma_pair(pair_of(y[8 * k + 2 * i], y[8 * k + 2 * i + 1]), r2, 0), e, f);
                                if (a.gate) {
                                    const __nv_bfloat162 plain = __floats2bfloat162_rn(e, f);
                                    if (c + 8 * k < o_end) none = __hfma2(plain, zero, none);
                                    const uint32_t z = ((const uint32_t*)at_stage(lane, k))[i];
                                    e *= sigmoid_for<bf16>(bf16_lo(z)) * a.out_scale;
                                    f *= sigmoid_for<bf16>(bf16_hi(z)) * a.out_scale;
                                }
                                x[i] = pack_bf16(e, f);
                                if (!a.gate && c + 8 * k < o_end) none = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&x[i]), zero, none);
                            }
                            *at_stage(lane, k) = make_uint4(x[0], x[1], x[2], x[3]);
                        }
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (to[k] >= 0 && col < o_end) *(uint4*)((bf16*)a.out + to[k] + col) = *at_stage((lane >> 1) + 16 * k, piece);
                        __syncwarp();
                    }
                    const float2 bad = __bfloat1622float2(none);
                    for (unsigned again = __ballot_sync(0xffffffffu, row < rows && !(bad.x == 0.f && bad.y == 0.f)); again; again &= again - 1) {
                        const int who = __ffs(again) - 1;
                        finish_again<bf16>(p, b, kv, __shfl_sync(0xffffffffu, tok, who), __shfl_sync(0xffffffffu, head, who), __shfl_sync(0xffffffffu, pos, who),
                                           o_begin, o_end);
                    }
                } else {
                    float* mine = p.part + slot * a.dv;
#pragma unroll 2
                    for (int c = o_begin; c < o_end; c += 8) {
                        int32_t y[8] = {};
                        if (any) {
                            tmem_ld8(tO + (uint32_t)c, y);
                            tmem_ld_wait();
                        }
                        if (row < rows)
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(mine + c), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]),
                                         "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7]) : "memory");
                        __syncwarp();
                    }
                    if (row < rows) p.ml[slot * 2 + half] = half ? l : m;
                }
            }
            if (any) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s.o_empty[g]));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && s.abort) *(volatile int*)p.error_flag = 1;
}

struct TileShape {
    int rows, box, seg, segv, k_slots, v_stages;
    size_t smem;
    TileShape(const zkfp_paged_attention_args& a)
    {
        const int group = a.heads / a.kv_heads;
        rows = group <= kTile ? kTile / group * group : 0;
        box = a.page < kTile ? a.page : kTile;
        seg = (a.d + 63) / 64;
        segv = (a.dv + 63) / 64;
        const size_t fixed = 1024 + ((sizeof(TileShared) + 15) & ~15) + plan_bytes(a.batch), segs = (kSharedMax - 1024 - fixed) / kSeg;
        v_stages = 3 * seg + 2 * segv <= (int)segs ? 2 : 1;
        const int left = (int)segs - 2 * seg - v_stages * segv;
        k_slots = left < kMaxKeySlots ? left : kMaxKeySlots;
        smem = fixed + kSeg * (size_t)(2 * seg + k_slots + v_stages * segv);
    }
};

// [size][heads][lines][pages], pieces of 64 columns of one head of `rows` lines of a page
bool pages_map(CUtensorMap* map, const void* base, int size, int heads, int page, long long pages, long long head, long long pos, long long stride,
               int rows)
{
    auto at_least = [](long long s, long long least) { return (uint64_t)(s > 0 ? s : least) * 2; };       // one head, line or page has no stride
    const uint64_t dims[4] = {(uint64_t)size, (uint64_t)heads, (uint64_t)page, (uint64_t)pages};
    const uint64_t strides[3] = {at_least(head, size), at_least(pos, size), at_least(stride, size)};
    const uint32_t box[4] = {64, 1, (uint32_t)rows, 1};
    return fp_tensor_map(map, base, 4, dims, strides, box);
}

bool key_maps(CUtensorMap* k, CUtensorMap* v, const zkfp_paged_attention_args& a, int rows)
{
    return pages_map(k, a.k, a.d, a.kv_heads, a.page, a.pages, a.k_head, a.k_pos, a.k_page, rows) &&
           pages_map(v, a.v, a.dv, a.kv_heads, a.page, a.pages, a.v_head, a.v_pos, a.v_page, rows);
}

// Tensor maps have no dimension that does not move on (a tensor expanded over heads, pages or tokens): the CUDA cores take those.
bool moves(long long n, long long stride) { return n == 1 || stride > 0; }
bool pages_move(const zkfp_paged_attention_args& a)
{
    return moves(a.kv_heads, a.k_head) && moves(a.kv_heads, a.v_head) && moves(a.page, a.k_pos) && moves(a.page, a.v_pos) && moves(a.pages, a.k_page) &&
           moves(a.pages, a.v_page);
}

}  // namespace

bool paged_stream_takes(const zkfp_paged_attention_args& a)
{
    return pages_move(a) && a.dtype == ZKFP_BF16 && a.d <= kStreamMost && a.dv <= kStreamMost && a.max_tokens * (a.heads / a.kv_heads) <= kStreamRows &&
           StreamShape(a).stages >= 2;
}

void paged_stream_shape(Paged& p)
{
    p.tile = kStreamRows;
    p.block = kStreamKeys;
    p.grid = 2 * fp_sm_count();
    p.over = kStreamOver;
    p.least = kStreamLeast;
}

template <int SEGK, int SEGV>
static int launch_stream(const Paged& p, const CUtensorMap& k, const CUtensorMap& v, const StreamShape& s, cudaStream_t st)
{
    ZKDS_CUDA(cudaFuncSetAttribute(paged_stream_kernel<SEGK, SEGV>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax - 1024));
    fp_launch(paged_stream_kernel<SEGK, SEGV>, dim3((unsigned)p.grid), dim3(kStreamWarps * 32), s.smem, st, k, v, p, s.box, s.stages);
    return fp_launched();
}

bool paged_tile_takes(const zkfp_paged_attention_args& a)
{
    if (a.dtype != ZKFP_BF16 || a.d > kTileMost || a.dv > kTileMost || !pages_move(a) || !moves(a.heads, a.q_head) || !moves(a.tokens, a.q_tok)) return false;
    const TileShape s(a);
    return s.rows > 0 && s.k_slots >= s.seg;
}

void paged_tile_shape(Paged& p)
{
    p.tile = 2 * TileShape(p.a).rows;
    p.block = kTile;
    p.grid = fp_sm_count();
    p.over = kTileOver;
    p.least = kTileLeast;
}

int launch_paged_tile(const Paged& p, cudaStream_t st)
{
    const zkfp_paged_attention_args& a = p.a;
    const TileShape s(a);
    TileParams t;
    t.p = p;
    t.rows = s.rows; t.box = s.box; t.seg = s.seg; t.segv = s.segv; t.k_slots = s.k_slots; t.v_stages = s.v_stages;
    t.scale_log2 = a.scale * kLog2e;
    CUtensorMap q, k, v;
    const uint64_t G = (uint64_t)p.group, head = (uint64_t)(a.q_head > 0 ? a.q_head : a.d) * 2;
    const uint64_t dims[4] = {(uint64_t)a.d, G, (uint64_t)a.kv_heads, (uint64_t)a.tokens};
    const uint64_t strides[3] = {head, head * G, a.q_tok > 0 ? (uint64_t)a.q_tok * 2 : head * G * a.kv_heads};
    const uint32_t box[4] = {64, (uint32_t)G, 1, (uint32_t)(s.rows / p.group)};
    if (!fp_tensor_map(&q, a.q, 4, dims, strides, box) || !key_maps(&k, &v, a, s.box)) return ZKDS_ERR_UNSUPPORTED;
    ZKDS_CUDA(cudaFuncSetAttribute(paged_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax - 1024));
    // more than half the shared memory: one CTA per SM, so the tensor-memory allocation never waits
    const size_t smem = s.smem < 120 * 1024 ? 120 * 1024 : s.smem;
    fp_launch(paged_tile_kernel, dim3((unsigned)p.grid), dim3(kTileThreads), smem, st, q, k, v, t);
    return fp_launched();
}

int launch_paged_stream(const Paged& p, cudaStream_t st)
{
    const StreamShape s(p.a);
    CUtensorMap k, v;
    if (!key_maps(&k, &v, p.a, s.box)) return ZKDS_ERR_UNSUPPORTED;
    if (s.segk == 1) return s.segv == 1 ? launch_stream<1, 1>(p, k, v, s, st) : launch_stream<1, 2>(p, k, v, s, st);
    return s.segv == 1 ? launch_stream<2, 1>(p, k, v, s, st) : launch_stream<2, 2>(p, k, v, s, st);
}

}  // namespace zkds
