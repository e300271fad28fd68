// A pool of pages: new keys and values to their pages (turned on the way), and copies of pages between one another.
#include <stdlib.h>
#include <string.h>

#include "float_common.cuh"
#include "float_paged.cuh"

namespace zkds {

namespace {

// ---- copies ------------------------------------------------------------------------------------------------------
// One launch copies up to kMoves pages in up to kBuffers buffers; the list travels in the launch's parameters, so there is
// no table to upload and none to keep alive.  A block moves 16 KB.  1500 pages of 256 KB in three buffers: 366 us, 6.4 TB/s, the rate of a plain
// copy; three pages of 148 KB in 24 buffers: 3.8 us.
constexpr int kMoves = 384, kBuffers = 32, kCopyThreads = 256, kCopyVecs = 4;
constexpr long long kCopyBytes = (long long)kCopyThreads * kCopyVecs * 16;

struct CopyList {
    char* base[kBuffers];
    long long stride[kBuffers];
    unsigned vecs[kBuffers];         // 16-byte pieces of a page
    int source[kMoves], target[kMoves];
};

__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const __grid_constant__ CopyList list)
{
    chain_enter();
    const int n = blockIdx.z, m = blockIdx.y;
    const unsigned first = blockIdx.x * (kCopyThreads * kCopyVecs) + threadIdx.x, vecs = list.vecs[n];
    const uint4* src = (const uint4*)(list.base[n] + list.source[m] * list.stride[n]);
    uint4* dst = (uint4*)(list.base[n] + list.target[m] * list.stride[n]);
    uint4 v[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
        if (first + i * kCopyThreads < vecs) v[i] = src[first + i * kCopyThreads];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
        if (first + i * kCopyThreads < vecs) dst[first + i * kCopyThreads] = v[i];
}

// every page inside every buffer, no target twice, none both source and target
bool moves_ok(const int* source, const int* target, long long moves, long long pages)
{
    unsigned char* seen = (unsigned char*)calloc((size_t)pages, 1);
    if (!seen) return false;
    bool ok = true;
    for (long long i = 0; i < moves && ok; ++i) {
        ok = source[i] >= 0 && source[i] < pages && target[i] >= 0 && target[i] < pages && !seen[target[i]];
        if (ok) seen[target[i]] = 1;
    }
    for (long long i = 0; i < moves && ok; ++i) ok = !seen[source[i]];
    free(seen);
    return ok;
}

// ---- heads into pages --------------------------------------------------------------------------------------------
// A block takes one row and every gridDim.y-th group of its heads: queries, keys, then values.  A head is cut into units: eight elements of
// adjacent pairs (which turn all or not at all, or some of them where the pairs end inside a unit), two times eight of pairs half a rotation apart, or
// single pairs where those do not lie on 16-byte pieces; what does not turn is copied, bit by bit.  A thread keeps its unit, and so its angles, from head
// to head, and has 64 bytes on their way at a time (single pairs: four of them).  Every element is read and written by one thread, so q_out may be q.
// Bytes bound it: two prompts of 4095 tokens, 128 + 2 x 16 heads of 128, move 0.68 GB in 125 us (one head at a time, angles loaded for each: 156); in
// halves, all or half of a head, 131 and 154, single pairs 391 (one at a time 485).  Units that choose pair by pair take 1 % longer, and are another kernel.
constexpr int kWriteThreads = 256;
enum { kAdjacent, kAdjacentSome, kApart, kSingle };

__device__ __forceinline__ void turn(float& a, float& b, float2 cs)
{
    const float u = a * cs.x - b * cs.y;
    b = b * cs.x + a * cs.y;
    a = u;
}

// eight elements as they lie in memory
template <typename T>
struct Eight {
    static constexpr int N = sizeof(T) / 2;
    uint4 v[N];
    __device__ __forceinline__ void load(const T* p)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void store(T* p) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const { load8(reinterpret_cast<const T*>(v), x); }
    __device__ __forceinline__ void put(const float (&x)[8]) { store8(reinterpret_cast<T*>(v), x); }
    // the first `pairs` adjacent pairs
    __device__ __forceinline__ void set(const float (&x)[8], int pairs)
    {
        Eight y;
        y.put(x);
        uint32_t *to = reinterpret_cast<uint32_t*>(v), *from = reinterpret_cast<uint32_t*>(y.v);
#pragma unroll
        for (int k = 0; k < 4 * N; ++k) to[k] = k / N < pairs ? from[k] : to[k];
    }
};

// Unit u of `heads` heads, from `src` to `dst`, heads `step` apart beginning with `first`.  cs: null where nothing turns.
template <typename T, int KIND>
__device__ __forceinline__ void turn_heads(const T* src, long long src_head, T* dst, long long dst_head, int u, int pairs, const float2* cs, int first,
                                           int step, int heads)
{
    if (KIND == kSingle) {
        constexpr int kAhead = 4;
        const bool two = u < pairs, turns = two && cs;
        const float2 t = turns ? cs[u] : make_float2(1.f, 0.f);
        for (int h0 = first; h0 < heads; h0 += kAhead * step) {
            T x[kAhead], y[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (h0 + i * step < heads) {
                    const T* from = src + (h0 + i * step) * src_head + u;
                    y[i] = from[pairs];
                    if (two) x[i] = from[0];
                }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (h0 + i * step < heads) {
                    T* to = dst + (h0 + i * step) * dst_head + u;
                    if (turns) {
                        float a = to_f32(x[i]), b = to_f32(y[i]);
                        turn(a, b, t);
                        x[i] = from_f32<T>(a);
                        y[i] = from_f32<T>(b);
                    }
                    if (two) to[0] = x[i];
                    to[pairs] = y[i];
                }
        }
        return;
    }
    constexpr bool kNext = KIND != kApart;             // pairs are adjacent
    constexpr int V = KIND == kApart ? 2 : 1, N = KIND == kApart ? 8 : 4, kAhead = 8 / (int)sizeof(T) / V;
    // pairs of this unit that turn; what does not is stored as it was loaded, bit by bit
    const int turns = cs ? min(max(pairs - N * u, 0), N) : 0;
    float2 t[N];
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = k < turns ? cs[N * u + k] : make_float2(1.f, 0.f);
    // behind the pairs a unit of two is the second of its pieces alone
    const bool both = kNext || 8 * u < pairs;
    const int at[2] = {8 * u, 8 * u + pairs};
    for (int h0 = first; h0 < heads; h0 += kAhead * step) {
        Eight<T> raw[kAhead][V];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (h0 + i * step < heads) {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v == V - 1 || both) raw[i][v].load(src + (h0 + i * step) * src_head + at[v]);
            }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (h0 + i * step < heads) {
                if (kNext || turns) {
                    float x[V][8];
#pragma unroll
                    for (int v = 0; v < V; ++v) raw[i][v].get(x[v]);
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        if (kNext) turn(x[0][2 * k & 7], x[0][(2 * k + 1) & 7], t[k]);
                        else turn(x[0][k], x[V - 1][k], t[k]);
                    }
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        if (kNext) raw[i][v].set(x[v], KIND == kAdjacentSome ? turns : turns == N ? 4 : 0);      // (a branch: 1 % longer)
                        else raw[i][v].put(x[v]);
                    }
                }
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v == V - 1 || both) raw[i][v].store(dst + (h0 + i * step) * dst_head + at[v]);
            }
    }
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kWriteThreads, 4)
write_pages_kernel(const __grid_constant__ zkfp_write_pages_args a, int shift, int* error_flag)
{
    chain_enter();
    const long long r = blockIdx.x;
    const int b = sequence_of_row(a.rows, (int)a.batch, r);
    if (b < 0) return;
    const int row0 = a.rows[b], n = a.rows[b + 1] - row0;
    const bool bad = row0 < 0 || row0 + (long long)n > a.tokens;
    if ((bad || a.lengths[b] < 0) && threadIdx.x == 0) *(volatile int*)(error_flag + 1) = 1;
    if (bad || row0 > r) return;
    const long long pos = (long long)a.lengths[b] - n + (r - row0);
    long long page = -1;
    if (pos >= 0) {
        if ((pos >> shift) < a.table_cols) page = a.table[b * a.table_ld + (pos >> shift)];
        if (page < 0 || page >= a.pages) {
            page = -1;
            if (threadIdx.x == 0) *(volatile int*)(error_flag + 1) = 1;
        }
    }
    const long long line = pos & (a.page - 1);
    const bool turned = a.cos_sin && pos >= 0 && pos < a.positions;
    const float2* cs = (const float2*)a.cos_sin + (turned ? pos * a.pairs : 0);
    // a row without angles is copied, in the units of the others
    const int pairs = turned || KIND == kApart || KIND == kSingle ? a.pairs : 0;
    const int units = KIND == kSingle ? a.d - a.pairs : (KIND == kApart ? a.d - a.pairs : a.d) / 8;
    const int per = units < kWriteThreads ? kWriteThreads / units : 1, step = per * gridDim.y, head = blockIdx.y * per + (int)threadIdx.x / units;
    if ((int)threadIdx.x < per * units || units > kWriteThreads)
        for (int u = threadIdx.x % units; u < units; u += kWriteThreads) {
            const int first = units > kWriteThreads ? blockIdx.y : head;
            if (a.q) turn_heads<T, KIND>((const T*)a.q + r * a.q_tok, a.q_head, (T*)a.q_out + r * a.qo_tok, a.qo_head, u, pairs, turned ? cs : nullptr, first, step, a.heads);
            if (page >= 0)
                turn_heads<T, KIND>((const T*)a.k + r * a.k_tok, a.k_head, (T*)a.k_pages + page * a.k_page + line * a.k_pos, a.kp_head, u, pairs,
                                    turned ? cs : nullptr, first, step, a.kv_heads);
            if (units <= kWriteThreads) break;
        }
    if (page < 0) return;
    const int vecs = a.dv / 8;
    for (int i = blockIdx.y * kWriteThreads + threadIdx.x; i < a.kv_heads * vecs; i += kWriteThreads * gridDim.y) {
        const int g = i / vecs, c = (i - g * vecs) * 8;
        Eight<T> x;
        x.load((const T*)a.v + r * a.v_tok + g * a.v_head + c);
        x.store((T*)a.v_pages + page * a.v_page + line * a.v_pos + g * a.vp_head + c);
    }
}

template <typename T>
int write_pages(const zkfp_write_pages_args& a, int* flag, cudaStream_t st)
{
    // few rows: their heads spread over more blocks
    const long long units = (a.q ? a.heads : 0) + a.kv_heads, most = (units * a.d / 8 + kWriteThreads - 1) / kWriteThreads;
    long long gy = (2ll * fp_sm_count() + a.tokens - 1) / a.tokens;
    gy = gy > most ? most : gy;
    const dim3 grid((unsigned)a.tokens, (unsigned)(gy < 1 ? 1 : gy)), block(kWriteThreads);
    const int shift = page_shift(a.page);
    if (!a.half && a.pairs & 3) fp_launch(write_pages_kernel<T, kAdjacentSome>, grid, block, 0, st, a, shift, flag);
    else if (!a.half) fp_launch(write_pages_kernel<T, kAdjacent>, grid, block, 0, st, a, shift, flag);
    else if (a.pairs & 7) fp_launch(write_pages_kernel<T, kSingle>, grid, block, 0, st, a, shift, flag);
    else fp_launch(write_pages_kernel<T, kApart>, grid, block, 0, st, a, shift, flag);
    return fp_launched();
}

}  // namespace

}  // namespace zkds

using namespace zkds;

extern "C" {

int zkfp_copy_pages(const zkfp_page_buffer* buffers, int n_buffers, const int* source, const int* target, long long moves,
                    void* stream)
{
    if (n_buffers < 0 || moves < 0 || (n_buffers && !buffers) || (moves && (!source || !target))) return ZKDS_ERR_ARG;
    if (!n_buffers || !moves) return ZKDS_OK;
    long long pages = 0x7fffffffll;
    for (int i = 0; i < n_buffers; ++i) {
        const zkfp_page_buffer& p = buffers[i];
        if (p.bytes == 0) continue;
        if (!p.base || p.bytes < 0 || p.stride < p.bytes || ((p.bytes | p.stride) & 15) || ((uintptr_t)p.base & 15) || p.pages <= 0 ||
            p.pages >= 0x7fffffffll)
            return ZKDS_ERR_ARG;
        if (p.bytes > 0x400000000ll) return ZKDS_ERR_UNSUPPORTED;
        pages = p.pages < pages ? p.pages : pages;
    }
    if (pages == 0x7fffffffll) return ZKDS_OK;         // nothing of any buffer
    if (!moves_ok(source, target, moves, pages)) return ZKDS_ERR_ARG;
    for (int b0 = 0; b0 < n_buffers; b0 += kBuffers) {
        CopyList list;
        const int nb = n_buffers - b0 < kBuffers ? n_buffers - b0 : kBuffers;
        long long most = 0;
        for (int i = 0; i < nb; ++i) {
            list.base[i] = (char*)buffers[b0 + i].base;
            list.stride[i] = buffers[b0 + i].stride;
            list.vecs[i] = (unsigned)(buffers[b0 + i].bytes / 16);
            most = buffers[b0 + i].bytes > most ? buffers[b0 + i].bytes : most;
        }
        const unsigned chunks = (unsigned)((most + kCopyBytes - 1) / kCopyBytes);
        if (!chunks) continue;
        for (long long m0 = 0; m0 < moves; m0 += kMoves) {
            const int nm = (int)(moves - m0 < kMoves ? moves - m0 : kMoves);
            memcpy(list.source, source + m0, sizeof(int) * nm);
            memcpy(list.target, target + m0, sizeof(int) * nm);
            fp_launch(copy_pages_kernel, dim3(chunks, (unsigned)nm, (unsigned)nb), dim3(kCopyThreads), 0, (cudaStream_t)stream, list);
            const int rc = fp_launched();
            if (rc != ZKDS_OK) return rc;
        }
    }
    return ZKDS_OK;
}

int zkfp_write_pages(const zkfp_write_pages_args* a, void* stream)
{
    if (!a || !a->k || !a->v || !a->k_pages || !a->v_pages || !a->table || !a->rows || !a->lengths || (a->q && !a->q_out) || a->tokens < 0 ||
        a->batch <= 0 || a->batch > 0x7fffffff || a->pages <= 0 || a->table_cols <= 0 || a->table_ld < a->table_cols ||
        page_shift(a->page) < 0 || (a->q && a->heads <= 0) || a->kv_heads <= 0 || a->d <= 0 || a->dv <= 0 || (a->d & 7) || (a->dv & 7) ||
        a->pairs < 0 || 2 * a->pairs > a->d || (a->cos_sin && a->positions < 0) || (unsigned)a->half > 1 || (unsigned)a->dtype > 1)
        return ZKDS_ERR_ARG;
    if ((a->q_tok | a->q_head | a->k_tok | a->k_head | a->v_tok | a->v_head | a->qo_tok | a->qo_head | a->k_page | a->k_pos | a->kp_head |
         a->v_page | a->v_pos | a->vp_head) & 7 ||
        ((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->k_pages | (uintptr_t)a->v_pages) & 15 ||
        (uintptr_t)a->cos_sin & 7)
        return ZKDS_ERR_ARG;
    if (a->tokens == 0) return ZKDS_OK;
    if (a->tokens > 0x7fffffffll || (long long)(a->heads + a->kv_heads) * a->d > 0x7fffffffll / 2) return ZKDS_ERR_UNSUPPORTED;
    int* flag = fp_error_flag();
    if (!flag) return ZKDS_ERR_WORKSPACE;
    return a->dtype == ZKFP_BF16 ? write_pages<bf16>(*a, flag, (cudaStream_t)stream) : write_pages<float>(*a, flag, (cudaStream_t)stream);
}

}  // extern "C"
