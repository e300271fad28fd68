// A pool of pages: new keys and values to their pages (turned on the way), and copies of pages between one another.
#include <stdlib.h>
#include <string.h>

#include "float_common.cuh"
#include "float_paged.cuh"

namespace zkds {

namespace {

// ---- copies ------------------------------------------------------------------------------------------------------
// One launch copies up to kMoves pages in up to kBuffers buffers; the list travels in the launch's parameters, so there is
// no table to upload and none to keep alive.  A block moves 16 KB.
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
// A block takes one row and every gridDim.y-th group of its heads: queries, keys, then values.  A head is cut into units: eight elements
// of adjacent pairs, two times eight of pairs half a rotation apart, or single pairs where those do not lie on
// 16-byte pieces; what does not turn is copied.  Every element is read and written by one thread, so q_out may be q.
constexpr int kWriteThreads = 256;

__device__ __forceinline__ void turn(float& a, float& b, float2 cs)
{
    const float u = a * cs.x - b * cs.y;
    b = b * cs.x + a * cs.y;
    a = u;
}

template <typename T>
__global__ void __launch_bounds__(kWriteThreads)
write_pages_kernel(const zkfp_write_pages_args a, int shift, int* error_flag)
{
    chain_enter();
    const long long r = blockIdx.x;
    const int b = sequence_of_row(a.rows, (int)a.batch, r);
    if (b < 0) return;
    const int row0 = a.rows[b], n = a.rows[b + 1] - row0;
    const long long pos = (long long)a.lengths[b] - n + (r - row0);
    long long page = -1;
    if (pos >= 0) {
        if ((pos >> shift) < a.table_cols) page = a.table[b * a.table_ld + (pos >> shift)];
        if (page < 0 || page >= a.pages) {
            page = -1;
            if (threadIdx.x == 0) *(volatile int*)error_flag = 1;
        }
    }
    const long long line = pos & (a.page - 1);
    const bool turned = a.cos_sin && pos >= 0 && pos < a.positions;
    const float2* cs = (const float2*)a.cos_sin + (turned ? pos * a.pairs : 0);
    const int pairs = turned ? a.pairs : 0, q_heads = a.q ? a.heads : 0;
    const bool single = a.half && (pairs & 7);
    const int units = single ? a.d - pairs : (a.half ? a.d - pairs : a.d) / 8;
    const int all = (q_heads + a.kv_heads) * units, step = kWriteThreads * gridDim.y;
    for (int i = blockIdx.y * kWriteThreads + threadIdx.x; i < all; i += step) {
        const int head = i / units, u = i - head * units, g = head - q_heads;
        if (g >= 0 && page < 0) continue;
        const T* src = g < 0 ? (const T*)a.q + r * a.q_tok + head * a.q_head : (const T*)a.k + r * a.k_tok + g * a.k_head;
        T* dst = g < 0 ? (T*)a.q_out + r * a.qo_tok + head * a.qo_head
                       : (T*)a.k_pages + page * a.k_page + line * a.k_pos + g * a.kp_head;
        if (single) {
            if (u < pairs) {
                float x = to_f32(src[u]), y = to_f32(src[u + pairs]);
                turn(x, y, cs[u]);
                dst[u] = from_f32<T>(x);
                dst[u + pairs] = from_f32<T>(y);
            } else {
                dst[u + pairs] = src[u + pairs];
            }
            continue;
        }
        float x[8];
        if (!a.half) {
            load8(src + u * 8, x);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (u * 4 + k < pairs) turn(x[2 * k], x[2 * k + 1], cs[u * 4 + k]);
            store8(dst + u * 8, x);
        } else if (u * 8 < pairs) {
            float y[8];
            load8(src + u * 8, x);
            load8(src + u * 8 + pairs, y);
#pragma unroll
            for (int k = 0; k < 8; ++k) turn(x[k], y[k], cs[u * 8 + k]);
            store8(dst + u * 8, x);
            store8(dst + u * 8 + pairs, y);
        } else {
            load8(src + u * 8 + pairs, x);
            store8(dst + u * 8 + pairs, x);
        }
    }
    if (page < 0) return;
    const int vecs = a.dv / 8;
    for (int i = blockIdx.y * kWriteThreads + threadIdx.x; i < a.kv_heads * vecs; i += step) {
        const int g = i / vecs, c = (i - g * vecs) * 8;
        float x[8];
        load8((const T*)a.v + r * a.v_tok + g * a.v_head + c, x);
        store8((T*)a.v_pages + page * a.v_page + line * a.v_pos + g * a.vp_head + c, x);
    }
}

template <typename T>
int write_pages(const zkfp_write_pages_args& a, int* flag, cudaStream_t st)
{
    // few rows: their heads spread over more blocks
    const long long units = (a.q ? a.heads : 0) + a.kv_heads, most = (units * a.d / 8 + kWriteThreads - 1) / kWriteThreads;
    long long gy = (2ll * fp_sm_count() + a.tokens - 1) / a.tokens;
    gy = gy > most ? most : gy;
    fp_launch(write_pages_kernel<T>, dim3((unsigned)a.tokens, (unsigned)(gy < 1 ? 1 : gy)), dim3(kWriteThreads), 0, st, a, page_shift(a.page), flag);
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
