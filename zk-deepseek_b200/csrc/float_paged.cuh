// What the kernels of a pool of pages share: page arithmetic and the place of a row in its batch.
#pragma once
#include "float_common.cuh"

namespace zkds {

// log2 of a page size; -1 where it is none (a power of two from 8 to 1024)
inline int page_shift(int page)
{
    for (int s = 3; s <= 10; ++s)
        if (page == 1 << s) return s;
    return -1;
}

// the sequence whose rows end behind row r, the same in every thread of the block, or -1 (all threads call it)
__device__ __forceinline__ int sequence_of_row(const int* rows, int batch, long long r)
{
    int b = 0;
    for (int base = 0; base < batch; base += blockDim.x) {
        const int i = base + (int)threadIdx.x;
        b += __syncthreads_count(i < batch && rows[i + 1] <= r);
    }
    return b < batch ? b : -1;
}

// ---- attention over pages: how the work is shared ----------------------------------------------------------------
// An item is a tile of query rows (token, head of a group, in this order) of one sequence and one key head; it takes a
// number of units: `over` for what an item costs by itself (queries, sums, results), then blocks of keys from the first that any
// of its rows sees to the last.  All units in the order sequence, key head, tile, block are cut into equal ranges, one
// per CTA (fewer CTAs where a range would have less than `least`), so that one long sequence among short ones, a prompt
// among decoding sequences or a single sequence all keep every SM busy, and neither grid nor scratch depends on
// lengths that only the device knows.  An item that one CTA takes whole goes straight to `out`; of one that is cut, every CTA
// leaves its sums, and paged_combine_kernel merges them in the order of the keys.  Results depend on lengths alone, not on timing.
constexpr int kPagedBatch = 1024;

// A division whose divisor the host knows, of 0 <= x < 2^31: the high bits of a product.  (The multiplier is 2^shift / divisor rounded up, its error
// times x below 2^shift.  What starts a launch is a chain of such steps, each of a CTA's few: with divisions one sequence took 13.2 us, without 12.8, 64 87.3 and 84.5, by themselves.)
struct Ratio {
    uint32_t mul;
    int shift;
    void set(int divisor)
    {
        int s = 0;
        while ((1 << s) < divisor) ++s;
        shift = 31 + s;
        mul = (uint32_t)(((1ull << shift) + divisor - 1) / divisor);
    }
    __device__ __forceinline__ int operator()(int x) const { return (int)(((uint64_t)(uint32_t)x * mul) >> shift); }
};

struct Paged {
    zkfp_paged_attention_args a;
    int shift, group, tile, block, grid, over, least;          // least: 2 to its power
    Ratio by_groups, by_tiles, by_blocks, by_heads;
    float* part;                     // [2 * grid][tile][dv] weighted sums; first the item that began in front of a CTA's
    float* ml;                       // [2 * grid][tile][2] maximum, sum        range, then the one that ends behind it
    int* cut;                        // [grid][8] the item that begins in a CTA's range and ends behind it
    int* error_flag;                 // two words, see fp_error_flag
};

// in dynamic shared memory: (batch + 1) units in front of each sequence, then its first row, rows and positions
struct Plan {
    long long* before;
    int *row0, *n, *len;
    __device__ __forceinline__ Plan(uint8_t* at, int batch)
    {
        before = (long long*)at;
        row0 = (int*)(before + batch + 1);
        n = row0 + batch;
        len = n + batch;
    }
};
inline size_t plan_bytes(long long batch) { return ((size_t)(batch + 1) * 8 + (size_t)batch * 12 + 15) & ~(size_t)15; }

__device__ __forceinline__ int by_group(const Paged& p, int x) { return p.by_groups(x); }

// the first position that a row at position i (which may be negative) sees
__device__ __forceinline__ int first_seen(const Paged& p, int i) { return p.a.window > 0 && i >= p.a.window ? i - p.a.window + 1 : 0; }

// blocks of keys that tile t of a sequence with n rows and len positions visits: first .. first + count - 1, one at least
__device__ __forceinline__ void tile_blocks(const Paged& p, int n, int len, int t, int& first, int& count)
{
    const int last_row = min((t + 1) * p.tile, n * p.group) - 1;
    const int i0 = len - n + by_group(p, t * p.tile), i1 = len - n + by_group(p, last_row);
    if (i1 < 0) { first = 0; count = 1; return; }
    first = p.by_blocks(first_seen(p, i0));
    count = p.by_blocks(i1) - first + 1;
}

__device__ __forceinline__ int tiles_of(const Paged& p, int n)
{
    const int rows = n * p.group;
    return p.by_tiles(rows + p.tile - 1);
}

__device__ __forceinline__ long long warp_sum64(long long v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// every thread of the block takes part; ends with a barrier
__device__ __forceinline__ void make_plan(const Paged& p, const Plan& s)
{
    const int batch = (int)p.a.batch, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const long long capacity = min(p.a.table_cols << p.shift, 0x7fffffffll);
    for (int base = warp * 32; base < batch; base += warps * 32) {
        const int b = base + lane;
        int n = 0, len = 0, row0 = 0;
        if (b < batch) {
            row0 = p.a.rows[b];
            const int row1 = p.a.rows[b + 1];
            len = p.a.lengths[b];
            n = row1 - row0;
            bool bad = len < 0 || len > capacity;
            len = len < 0 ? 0 : len > capacity ? (int)capacity : len;
            if (row0 < 0 || row1 < row0 || row1 > p.a.tokens) { n = 0; bad = true; }
            if (bad) *(volatile int*)(p.error_flag + 1) = 1;
        }
        const int tiles = tiles_of(p, n);
        long long units = 0;
        if (tiles <= 8)
            for (int t = 0; t < tiles; ++t) {
                int first, count;
                tile_blocks(p, n, len, t, first, count);
                units += count + p.over;
            }
        for (unsigned left = __ballot_sync(0xffffffffu, tiles > 8); left; left &= left - 1) {
            const int who = __ffs(left) - 1, nn = __shfl_sync(0xffffffffu, n, who), ll = __shfl_sync(0xffffffffu, len, who);
            long long sum = 0;
            for (int t = lane; t < tiles_of(p, nn); t += 32) {
                int first, count;
                tile_blocks(p, nn, ll, t, first, count);
                sum += count + p.over;
            }
            sum = warp_sum64(sum);
            if (lane == who) units = sum;
        }
        if (b < batch) {
            s.row0[b] = row0;
            s.n[b] = n;
            s.len[b] = len;
            s.before[b + 1] = units * p.a.kv_heads;
        }
    }
    __syncthreads();
    if (warp == 0) {
        long long total = 0;
        for (int base = 0; base < batch; base += 32) {
            const int b = base + lane;
            long long v = b < batch ? s.before[b + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long w = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += w;
            }
            if (b < batch) s.before[b + 1] = total + v;
            total += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) s.before[0] = 0;
    }
    __syncthreads();
}

// CTAs that share the units, how many each, and how many CTAs one more
struct Share {
    int ctas, more;
    long long each;
    __device__ __forceinline__ Share(const Paged& p, long long units)
    {
        const long long most = units >> p.least;
        ctas = most < 1 ? 1 : most < p.grid ? (int)most : p.grid;
        each = units < 0x80000000ll ? (uint32_t)units / (uint32_t)ctas : units / ctas;
        more = (int)(units - each * ctas);
    }
    __device__ __forceinline__ long long begin(int cta) const { return cta * each + min(cta, more); }
    // the first CTA whose range begins at unit u or behind it
    __device__ __forceinline__ int behind(long long u) const
    {
        const long long longer = more * (each + 1);
        const long long by = u <= longer ? each + 1 : each, in = (u <= longer ? u : u - longer) + by - 1;
        return (u <= longer ? 0 : more) + (in < 0x80000000ll ? (int)((uint32_t)in / (uint32_t)by) : (int)(in / by));
    }
};

// one item and the part of it that starts at unit u; whole warps walk, every warp by itself
struct Walk {
    int b, kv, t, tiles;             // sequence, key head, tile
    int first, count, at;            // blocks of the item, and which of its units (those for itself in front) u is
    int row0, n, len;

    __device__ __forceinline__ void sequence(const Paged& p, const Plan& s)
    {
        row0 = s.row0[b]; n = s.n[b]; len = s.len[b];
        tiles = tiles_of(p, n);
    }
    __device__ __forceinline__ void locate(const Paged& p, const Plan& s, long long u)
    {
        int lo = 0, hi = (int)p.a.batch;               // before[lo] <= u < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s.before[mid] <= u) lo = mid;
            else hi = mid;
        }
        b = lo;
        sequence(p, s);
        const long long mine = s.before[b + 1] - s.before[b], in = u - s.before[b];
        const long long per = mine < 0x80000000ll ? p.by_heads((int)mine) : mine / p.a.kv_heads;
        kv = p.a.kv_heads == 1 ? 0 : (int)(mine < 0x80000000ll ? (uint32_t)in / (uint32_t)per : in / per);
        long long rest = in - kv * per;
        const int lane = threadIdx.x & 31;
        for (int t0 = 0;; t0 += 32) {                  // ends: rest < per, the sum of all tiles
            int f = 0, c = -p.over;
            if (t0 + lane < tiles) tile_blocks(p, n, len, t0 + lane, f, c);
            int sum = c + p.over;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int w = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += w;
            }
            const unsigned past = __ballot_sync(0xffffffffu, sum > rest);
            if (past || t0 + 32 >= tiles) {
                const int who = past ? __ffs(past) - 1 : 31;
                t = t0 + who;
                at = (int)rest - __shfl_sync(0xffffffffu, sum - c - p.over, who);
                first = __shfl_sync(0xffffffffu, f, who);
                count = __shfl_sync(0xffffffffu, c, who);
                return;
            }
            rest -= __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    // units of the item from here on
    __device__ __forceinline__ int left(const Paged& p) const { return p.over + count - at; }
    // blocks of the item, from its first, in front of this unit and of the one `taken` further on
    __device__ __forceinline__ int begin(const Paged& p) const { return max(at - p.over, 0); }
    __device__ __forceinline__ int end(const Paged& p, int taken) const { return max(at + taken - p.over, 0); }
    __device__ __forceinline__ void next(const Paged& p, const Plan& s)
    {
        at = 0;
        if (++t == tiles) {
            t = 0;
            if (++kv == p.a.kv_heads) {
                kv = 0;
                do ++b;
                while (b < p.a.batch && s.before[b + 1] == s.before[b]);
                if (b == p.a.batch) return;
                sequence(p, s);
            }
        }
        if (tiles > 1 || kv == 0) tile_blocks(p, n, len, t, first, count);      // else as for the key head in front
    }
};

// What paged_combine_kernel has to know of the item whose first block CTA `cta` takes and whose last one it does not: in how many
// parts it was taken, 0 for none.  `end`: the unit behind the item's last.  One thread writes it, of every CTA of the grid.
__device__ __forceinline__ void no_cut(const Paged& p, int cta) { p.cut[cta * 8] = 0; }
__device__ __forceinline__ void write_cut(const Paged& p, int cta, const Share& share, const Walk& w, long long end)
{
    int4* to = (int4*)(p.cut + cta * 8);
    to[0] = make_int4(share.behind(end) - cta, w.b, w.kv, w.t);
    to[1] = make_int4(w.row0, w.n, w.len, 0);
}

// page of position j, or -1
__device__ __forceinline__ long long page_of(const Paged& p, int b, int j)
{
    const long long page = p.a.table[b * p.a.table_ld + (j >> p.shift)];
    return page >= 0 && page < p.a.pages ? page : -1;
}

// ---- a row by itself ---------------------------------------------------------------------------------------------
// The tiles multiply weights of zero with whatever values stand at positions that a row does not see.  Where that
// is an infinity or a NaN (another row's), or where a visible score is NaN, the row's sums are not finite, and the row is
// taken once more from the definition, visible positions alone.  A warp takes 32 keys at a time, a lane one key, then a lane every
// 32nd column.  o[k]: column lane + 32 k.
template <typename T>
__device__ __noinline__ void attend_row(const Paged& p, int b, int kv, int token, int head, int pos, float (&o)[8])
{
    const int lane = threadIdx.x & 31;
    const T* q = (const T*)p.a.q + (long long)token * p.a.q_tok + head * p.a.q_head;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
    for (int j0 = first_seen(p, pos); j0 <= pos; j0 += 32) {
        const int j = j0 + lane;
        const long long page = j <= pos ? page_of(p, b, j) : -1;
        float s = 0.f;
        if (page >= 0) {
            const T* key = (const T*)p.a.k + page * p.a.k_page + (j & (p.a.page - 1)) * p.a.k_pos + kv * p.a.k_head;
            for (int c = 0; c < p.a.d; c += 8) {
                float x[8], y[8];
                load8(q + c, x);
                load8(key + c, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(x[i], y[i], s);
            }
            s *= p.a.scale;
        }
        const float m_new = fmaxf(m, warp_max(page >= 0 ? s : -INFINITY));
        const float f = m == m_new ? 1.f : expf(m - m_new);
        const float e = page < 0 || (s == -INFINITY && m_new == -INFINITY) ? 0.f : expf(s - m_new);
        l = l * f + warp_sum(e);
        m = m_new;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] *= f;
        for (int i = 0; i < 32 && j0 + i <= pos; ++i) {
            const float w = __shfl_sync(0xffffffffu, e, i);
            const long long at = __shfl_sync(0xffffffffu, page, i);
            if (at < 0) continue;
            const T* value = (const T*)p.a.v + at * p.a.v_page + ((j0 + i) & (p.a.page - 1)) * p.a.v_pos + kv * p.a.v_head;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (lane + 32 * k < p.a.dv) o[k] = fmaf(w, to_f32(value[lane + 32 * k]), o[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] /= l;
}

// The row's columns from `begin` to `end` in `out`, from the definition
template <typename T>
__device__ __noinline__ void finish_again(const Paged& p, int b, int kv, int token, int head, int pos, int begin, int end)
{
    float x[8];
    attend_row<T>(p, b, kv, token, head, pos, x);
    const int lane = threadIdx.x & 31;
    T* out = (T*)p.a.out + (long long)token * p.a.o_tok + head * p.a.o_head;
    const T* gate = p.a.gate ? (const T*)p.a.gate + (long long)token * p.a.gate_tok + head * p.a.gate_head : nullptr;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int c = lane + 32 * k;
        if (c < begin || c >= end) continue;
        if (gate) x[k] *= sigmoid_f(to_f32(gate[c])) * p.a.out_scale;
        out[c] = from_f32<T>(x[k]);
    }
}

__device__ __forceinline__ void load4(const float* p, float (&v)[4])
{
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void load4(const bf16* p, float (&v)[4])
{
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y);
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(bf16* p, const float (&v)[4])
{
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
}

// A warp finishes a row: x[k] are the weighted sums of columns 4 lane + 128 k and the three behind, l is the sum of the weights.
template <typename T, int K>
__device__ __forceinline__ void finish_row(const Paged& p, const Walk& w, int row, float (&x)[K][4], float l)
{
    const int lane = threadIdx.x & 31, in_seq = by_group(p, row), head = w.kv * p.group + row - in_seq * p.group;
    const int token = w.row0 + in_seq, pos = w.len - w.n + in_seq;
    T* out = (T*)p.a.out + (long long)token * p.a.o_tok + head * p.a.o_head;
    const T* gate = p.a.gate ? (const T*)p.a.gate + (long long)token * p.a.gate_tok + head * p.a.gate_head : nullptr;
    float none = 0.f;                                  // stays zero where everything is finite
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = 4 * lane + 128 * k;
        if (c >= p.a.dv) break;
        float z[4];
        if (gate) load4(gate + c, z);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[k][i] = pos < 0 ? 0.f : x[k][i] / l;
            none = fmaf(x[k][i], 0.f, none);
            if (gate) x[k][i] *= sigmoid_for<T>(z[i]) * p.a.out_scale;
        }
    }
    if (!__all_sync(0xffffffffu, none == 0.f)) {
        finish_again<T>(p, w.b, w.kv, token, head, pos, 0, p.a.dv);
        return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (4 * lane + 128 * k < p.a.dv) store4(out + 4 * lane + 128 * k, x[k]);
}

// ---- kernels on the tensor cores (float_paged_tc.cu): whether they take a call, their tile and grid, and the launch -----
bool paged_stream_takes(const zkfp_paged_attention_args& a);
void paged_stream_shape(Paged& p);
int launch_paged_stream(const Paged& p, cudaStream_t st);
bool paged_tile_takes(const zkfp_paged_attention_args& a);
void paged_tile_shape(Paged& p);
int launch_paged_tile(const Paged& p, cudaStream_t st);

}  // namespace zkds
