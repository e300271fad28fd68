// Attention of new tokens over pages: the kernels of CUDA cores (float32, and what the tensor cores do not take) and
// the one that merges what the CTAs of a cut item leave.  How the work is shared is in float_paged.cuh.
#include "float_paged.cuh"
#include "tcgen05.cuh"

namespace zkds {

namespace {

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- CUDA cores, few rows of bfloat16 ------------------------------------------------------------------------------
// For what the tensor cores do not take (heads beyond 128, tensors that were expanded): tiles of 16 rows over blocks of 64 keys, all in shared
// memory, sums of a row in registers: a thread holds eight columns of up to four rows.  Loads and products take turns, which bounds it.
constexpr int kPlainRows = 16, kPlainKeys = 64, kPlainThreads = 128, kPlainMost = 256;

template <typename T>
struct PlainShape {
    int kpitch;
    size_t smem;
    PlainShape(const zkfp_paged_attention_args& a)
    {
        kpitch = a.d + 16 / (int)sizeof(T);            // rows shifted by one 16-byte piece: no bank conflicts
        smem = plan_bytes(a.batch) + (size_t)kPlainKeys * (kpitch + a.dv) * sizeof(T) +
               sizeof(float) * ((size_t)kPlainRows * (a.d + a.dv) + kPlainRows * kPlainKeys + 3 * kPlainRows);
    }
};

template <typename T>
__global__ void __launch_bounds__(kPlainThreads)
paged_plain_kernel(const __grid_constant__ Paged p, int kpitch)
{
    chain_enter();
    extern __shared__ __align__(16) uint8_t sm[];
    const zkfp_paged_attention_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, d = a.d, dv = a.dv, vd = d / 8, vv = dv / 8, batch = (int)a.batch;
    const Plan plan(sm, batch);
    T* Ks = (T*)(sm + (((size_t)(batch + 1) * 8 + (size_t)batch * 12 + 15) & ~(size_t)15));
    T* Vs = Ks + kPlainKeys * kpitch;
    float* Q = (float*)(Vs + kPlainKeys * dv);
    float* O = Q + kPlainRows * d;
    float* P = O + kPlainRows * dv;
    float* M = P + kPlainRows * kPlainKeys;
    float *L = M + kPlainRows, *F = L + kPlainRows;
    make_plan(p, plan);
    const long long units = plan.before[batch];
    const Share share(p, units);
    const int cta = blockIdx.x;
    if (tid == 0) no_cut(p, cta);
    if (cta >= share.ctas || units == 0) return;
    const long long u1 = share.begin(cta + 1);
    long long u = share.begin(cta);
    Walk w;
    for (w.locate(p, plan, u); u < u1; w.next(p, plan)) {
        const int taken = (int)min((long long)w.left(p), u1 - u), j_begin = w.begin(p), j_end = w.end(p, taken);
        const long long end = u + w.left(p);
        u += taken;
        if (j_begin == j_end) continue;
        const bool whole = j_begin == 0 && j_end == w.count;
        if (tid == 0 && j_begin == 0 && !whole) write_cut(p, cta, share, w, end);
        const int slot = 2 * cta + (j_begin == 0 ? 1 : 0), row0 = w.t * kPlainRows, rows = min(kPlainRows, w.n * p.group - row0);
        __syncthreads();
        for (int i = tid; i < kPlainRows * vd; i += kPlainThreads) {
            const int r = i / vd, c = (i - r * vd) * 8;
            float x[8] = {};
            if (r < rows) {
                const int t = by_group(p, row0 + r), h = w.kv * p.group + row0 + r - t * p.group;
                load8((const T*)a.q + (long long)(w.row0 + t) * a.q_tok + h * a.q_head + c, x);
            }
            store8(Q + r * d + c, x);
        }
        if (tid < kPlainRows) { M[tid] = -INFINITY; L[tid] = 0.f; }
        float acc[4][8] = {};
        for (int j = j_begin; j < j_end; ++j) {
            const int k0 = (w.first + j) * kPlainKeys, nk = min(kPlainKeys, w.len - k0);
            __syncthreads();                           // the block in front is done with keys, values and weights
            for (int i = tid; i < kPlainKeys * (vd + vv); i += kPlainThreads) {
                const int r = i / (vd + vv), c = i - r * (vd + vv);
                const long long page = r < nk ? page_of(p, w.b, k0 + r) : -1;
                if (r < nk && page < 0) *(volatile int*)(p.error_flag + 1) = 1;
                const long long line = (k0 + r) & (a.page - 1);
                const T* src = c < vd ? (const T*)a.k + page * a.k_page + line * a.k_pos + w.kv * a.k_head + c * 8
                                      : (const T*)a.v + page * a.v_page + line * a.v_pos + w.kv * a.v_head + (c - vd) * 8;
                T* dst = c < vd ? Ks + r * kpitch + c * 8 : Vs + r * dv + (c - vd) * 8;
#pragma unroll
                for (int q = 0; q < (int)sizeof(T) / 2; ++q)
                    reinterpret_cast<uint4*>(dst)[q] = page >= 0 ? reinterpret_cast<const uint4*>(src)[q] : make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
            // scores: a thread takes one key and four rows
            for (int i = tid; i < kPlainKeys * (kPlainRows / 4); i += kPlainThreads) {
                const int key = i % kPlainKeys, r = i / kPlainKeys * 4;
                if (r >= rows) continue;
                float s[4] = {};
                for (int c = 0; c < d; c += 8) {
                    float k8[8];
                    load8(Ks + key * kpitch + c, k8);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float q8[8];
                        load8(Q + (r + q) * d + c, q8);
#pragma unroll
                        for (int e = 0; e < 8; ++e) s[q] = fmaf(q8[e], k8[e], s[q]);
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) P[(r + q) * kPlainKeys + key] = s[q];
            }
            __syncthreads();
            // softmax of the block, a warp per row
            for (int r = tid >> 5; r < rows; r += kPlainThreads / 32) {
                const int pos = w.len - w.n + by_group(p, row0 + r);
                float s[kPlainKeys / 32], m = M[r];
                const float m_old = m;
#pragma unroll
                for (int i = 0; i < kPlainKeys / 32; ++i) {
                    const int key = k0 + i * 32 + lane;
                    const bool seen = key <= pos && (a.window <= 0 || pos - key < a.window);
                    s[i] = seen ? P[r * kPlainKeys + i * 32 + lane] * a.scale : -INFINITY;
                    m = fmaxf(m, s[i]);
                }
                m = warp_max(m);
                float l = 0.f;
#pragma unroll
                for (int i = 0; i < kPlainKeys / 32; ++i) {
                    const float e = s[i] == -INFINITY ? 0.f : expf(s[i] - m);
                    P[r * kPlainKeys + i * 32 + lane] = e;
                    l += e;
                }
                l = warp_sum(l);
                if (lane == 0) {
                    const float f = m_old == -INFINITY ? 0.f : expf(m_old - m);
                    M[r] = m;
                    L[r] = L[r] * f + l;
                    F[r] = f;
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = tid + k * kPlainThreads, r = i / vv, c = (i - r * vv) * 8;
                if (r >= rows) break;
                const float f = F[r];
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[k][e] *= f;
#pragma unroll 4
                for (int key = 0; key < kPlainKeys; ++key) {
                    float v8[8];
                    load8(Vs + key * dv + c, v8);
                    const float e = P[r * kPlainKeys + key];
#pragma unroll
                    for (int q = 0; q < 8; ++q) acc[k][q] = fmaf(e, v8[q], acc[k][q]);
                }
            }
        }
        float* to = whole ? O : p.part + (long long)slot * p.tile * dv;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = tid + k * kPlainThreads, r = i / vv, c = (i - r * vv) * 8;
            if (r < rows) store8(to + r * dv + c, acc[k]);
        }
        if (whole) {
            __syncthreads();
            for (int r = tid >> 5; r < rows; r += kPlainThreads / 32) {
                float x[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (4 * lane + 128 * k < dv) load4(O + r * dv + 4 * lane + 128 * k, x[k]);
                finish_row<T>(p, w, row0 + r, x, L[r]);
            }
        } else if (tid < rows) {
            p.ml[((long long)slot * p.tile + tid) * 2] = M[tid];
            p.ml[((long long)slot * p.tile + tid) * 2 + 1] = L[tid];
        }
    }
}

// ---- CUDA cores, few rows of float32 -------------------------------------------------------------------------------
// Up to R rows (4 or 8) per key head, so that the bytes of keys and values are the bound.  A warp works by itself, on every fourth stretch of 16
// keys, which it asks for line by line; as in the kernel below, the four lanes that share rows and keys deal the head out among themselves in pairs of
// elements and hand each other their sums, weights pass through shared memory, the next stretch's keys are on their way under the softmax and the second
// product and its values under the next scores.  The warps' sums meet at the end of the item.
// One new token of 1, 16, 64 sequences of up to 1024 positions, 16 heads of 128 over 4: 12, 14, 20 us (tiles of eight rows instead of four 14, 17, 25;
// the kernel above, all warps on one block, 27, 29, 56).  Eight sequences with 6 and 8 tokens each, 24 and 32 rows: 19 and 24 us, the kernel below 22
// and 24, so that 24 rows is where that one begins.
constexpr int kFewRows = 24, kFewWarps = 4, kFewKeys = 16, kFewBlock = kFewWarps * kFewKeys, kFewThreads = kFewWarps * 32, kFewPitch = kFewKeys + 4;

template <int R>
struct FewShared {
    uint64_t full[kFewWarps][2];                       // keys, values
    uint64_t q_full;
    float m[kFewWarps][R], l[kFewWarps][R];
    __align__(16) float weights[kFewWarps][R][kFewPitch];
    int gave_up;
};

template <int R>
size_t few_bytes(const zkfp_paged_attention_args& a)
{
    return plan_bytes(a.batch) + sizeof(float) * ((size_t)kFewBlock * (a.d + 4 + a.dv) + (size_t)R * a.d) + sizeof(FewShared<R>);
}

template <int R, int PAIRS>
__global__ void __launch_bounds__(kFewThreads, PAIRS <= 4 ? 3 : 2)
paged_few_kernel(const __grid_constant__ Paged p)
{
    extern __shared__ __align__(16) uint8_t sm[];
    const zkfp_paged_attention_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = a.d, dv = a.dv, kpitch = d + 4, batch = (int)a.batch;
    constexpr int kEach = R / 4;                       // rows of a lane behind the scores
    const Plan plan(sm, batch);
    float* ring = (float*)(sm + (((size_t)(batch + 1) * 8 + (size_t)batch * 12 + 15) & ~(size_t)15));
    float* K = ring + warp * kFewKeys * (kpitch + dv);                                                         // [key][kpitch]; at the end [row][dv]
    float* V = K + kFewKeys * kpitch;                                                                          // [key][dv]
    float* Q = ring + kFewBlock * (kpitch + dv);                                                               // [row][d]
    FewShared<R>& sh = *(FewShared<R>*)(Q + R * d);
    if (tid == 0) {
        for (int i = 0; i < kFewWarps; ++i) {
            mbar_init(smem_u32(&sh.full[i][0]), kFewKeys);
            mbar_init(smem_u32(&sh.full[i][1]), kFewKeys);
        }
        mbar_init(smem_u32(&sh.q_full), R);
        sh.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_enter();                                     // barriers touch nobody else
    make_plan(p, plan);
    const long long units = plan.before[batch];
    const Share share(p, units);
    const int cta = blockIdx.x;
    if (tid == 0) no_cut(p, cta);
    if (cta >= share.ctas || units == 0) return;
    const long long u1 = share.begin(cta + 1);
    long long u = share.begin(cta);
    // scores: keys kg + 8 e, pairs sp, sp + 4, ... of the head; then rows r0 and on.  Values: column pairs cl + 16 k, keys 8 i + 4 kh + 0 .. 3.
    const int kg = lane & 7, sp = lane >> 3, r0 = R / 2 * (sp & 1) + kEach * (sp >> 1), cl = lane & 15, kh = lane >> 4;
    const int line_of = lane & (kFewKeys - 1);
    const bool values = lane >= kFewKeys;              // which lines this lane asks for
    const float scale = a.scale * 1.4426950408889634f;
    int column[PAIRS];                                 // behind the last one: that one again, without a branch, and not stored
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) column[k] = min(32 * k + 2 * cl, dv - 2);
    uint32_t phase = 0, q_phase = 0;
    bool ok = true;
    Walk w;
    for (w.locate(p, plan, u); u < u1; w.next(p, plan)) {
        const int taken = (int)min((long long)w.left(p), u1 - u), j_begin = w.begin(p), j_end = w.end(p, taken);
        const long long end = u + w.left(p);
        u += taken;
        if (j_begin == j_end) continue;
        const bool whole = j_begin == 0 && j_end == w.count;
        if (tid == 0 && j_begin == 0 && !whole) write_cut(p, cta, share, w, end);
        const int slot = 2 * cta + (j_begin == 0 ? 1 : 0), row0 = w.t * R, rows = min(R, w.n * p.group - row0);
        const float* from = values ? (const float*)a.v + w.kv * a.v_head : (const float*)a.k + w.kv * a.k_head;
        const long long page_step = values ? a.v_page : a.k_page, line_step = values ? a.v_pos : a.k_pos;
        float* to = values ? V + line_of * dv : K + line_of * kpitch;
        const int size = values ? dv : d;
        const uint32_t bar = smem_u32(&sh.full[warp][values]);
        // the position of this lane's line of block j, its page, looked up a stretch ahead and looked at when it is needed, and the request
        auto key_of = [&](int j) { return (w.first + j) * kFewBlock + warp * kFewKeys + line_of; };
        auto find = [&](int j) { return j < j_end && key_of(j) < w.len ? a.table[w.b * a.table_ld + (key_of(j) >> p.shift)] : 0; };
        auto request = [&](int j, int page) {
            const int k = key_of(j);
            const bool there = k < w.len && page >= 0 && page < a.pages;
            if (k < w.len && !there) *(volatile int*)(p.error_flag + 1) = 1;
            if (there) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // zeros that the line held
                mbar_expect_tx(bar, size * 4);
                bulk_load(smem_u32(to), from + page * page_step + (k & (a.page - 1)) * line_step, size * 4, bar);
            } else {
                for (int c = 0; c < size; c += 4) *(float4*)(to + c) = make_float4(0.f, 0.f, 0.f, 0.f);
                mbar_arrive(bar);
            }
        };
        request(j_begin, find(j_begin));
        int ahead = find(j_begin + 1);
        if (tid < R) {
            // rows behind the last hold what they held, and nothing reads their results
            const int t = by_group(p, row0 + tid), h = w.kv * p.group + row0 + tid - t * p.group;
            mbar_expect_tx(smem_u32(&sh.q_full), tid < rows ? d * 4 : 0);
            if (tid < rows) bulk_load(smem_u32(Q + tid * d), (const float*)a.q + (long long)(w.row0 + t) * a.q_tok + h * a.q_head, d * 4, smem_u32(&sh.q_full));
        }
        __syncwarp();
        int pos[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) pos[i] = r0 + i < rows ? w.len - w.n + by_group(p, row0 + r0 + i) : -1;
        const int all_lo = first_seen(p, pos[kEach - 1]);
        float m[kEach], l[kEach];
        uint64_t acc[R][PAIRS];
#pragma unroll
        for (int i = 0; i < kEach; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) acc[i][k] = 0;
        if (ok) ok = mbar_wait_warp(smem_u32(&sh.q_full), q_phase, &sh.gave_up);
        q_phase ^= 1u;
        for (int j = j_begin; j < j_end; ++j) {
            const int k0 = (w.first + j) * kFewBlock + warp * kFewKeys;
            float s[R][2] = {};
            if (ok) ok = mbar_wait_warp(smem_u32(&sh.full[warp][0]), phase, &sh.gave_up);
#pragma unroll 2
            for (int c = 2 * sp; c < d; c += 8) {
                const float2 ka = *(const float2*)(K + kg * kpitch + c), kb = *(const float2*)(K + (kg + 8) * kpitch + c);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float2 q = *(const float2*)(Q + i * d + c);
                    s[i][0] = fmaf(q.y, ka.y, fmaf(q.x, ka.x, s[i][0]));
                    s[i][1] = fmaf(q.y, kb.y, fmaf(q.x, kb.x, s[i][1]));
                }
            }
            __syncwarp();                              // the keys have been read
            if (j + 1 < j_end && !values) request(j + 1, ahead);
            __syncwarp();
            float h[R / 2][2], v[kEach][2], top[kEach], f[kEach];
#pragma unroll
            for (int i = 0; i < R / 2; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) h[i][e] = (sp & 1 ? s[i + R / 2][e] : s[i][e]) + __shfl_xor_sync(0xffffffffu, sp & 1 ? s[i][e] : s[i + R / 2][e], 8);
#pragma unroll
            for (int i = 0; i < kEach; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) v[i][e] = (sp & 2 ? h[i + kEach][e] : h[i][e]) + __shfl_xor_sync(0xffffffffu, sp & 2 ? h[i][e] : h[i + kEach][e], 16);
            const bool edge = pos[kEach - 1] < 0 || k0 + kFewKeys - 1 > pos[0] || k0 < all_lo;
            float changed = 0.f;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = k0 + kg + 8 * e;
                    v[i][e] = edge && !(key <= pos[i] && (a.window <= 0 || pos[i] - key < a.window)) ? -INFINITY : v[i][e] * scale;
                }
                top[i] = fmaxf(v[i][0], v[i][1]);
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
                top[i] = fmaxf(top[i], m[i]);
                const float sub = top[i] == -INFINITY ? 0.f : top[i];
                f[i] = exp2_approx(m[i] - sub);
                changed += f[i] != 1.f;
                m[i] = top[i];
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    v[i][e] = exp2_approx(v[i][e] - sub);
                    sum += v[i][e];
                    sh.weights[warp][r0 + i][kg + 8 * e] = v[i][e];
                }
                l[i] = l[i] * f[i] + sum;              // of this lane's keys
            }
            if (__any_sync(0xffffffffu, changed != 0.f)) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const uint64_t f2 = twice(__shfl_sync(0xffffffffu, f[i % kEach], 8 * (i / (R / 2)) + 16 * (i % (R / 2) / kEach)));
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) {
                        uint64_t y = 0;
                        fma2(y, acc[i][k], f2);
                        acc[i][k] = y;
                    }
                }
            }
            __syncwarp();
            if (ok) ok = mbar_wait_warp(smem_u32(&sh.full[warp][1]), phase, &sh.gave_up);
            phase ^= 1u;
#pragma unroll
            for (int key = 0; key < kFewKeys; key += 8) {
                float x[R][4];
#pragma unroll
                for (int i = 0; i < R; ++i) load4(&sh.weights[warp][i][key + 4 * kh], x[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) {
                        const uint64_t y = *(const uint64_t*)(V + (key + 4 * kh + e) * dv + column[k]);
#pragma unroll
                        for (int i = 0; i < R; ++i) fma2(acc[i][k], y, twice(x[i][e]));
                    }
            }
            __syncwarp();                              // the values have been read, and the weights
            if (j + 1 < j_end && values) request(j + 1, ahead);
            __syncwarp();
            ahead = find(j + 2);
        }
        // the warps' sums, each in the place of its keys
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
            if (kg == 0) {
                sh.m[warp][r0 + i] = m[i];
                sh.l[warp][r0 + i] = l[i];
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                const uint64_t y = __shfl_xor_sync(0xffffffffu, acc[i][k], 16);
                const float x0 = __uint_as_float((uint32_t)acc[i][k]) + __uint_as_float((uint32_t)y);
                const float x1 = __uint_as_float((uint32_t)(acc[i][k] >> 32)) + __uint_as_float((uint32_t)(y >> 32));
                if (kh == (i & 1) && 32 * k + 2 * cl < dv) *(float2*)(K + i * dv + 32 * k + 2 * cl) = make_float2(x0, x1);
            }
        __syncthreads();
        for (int i = warp; i < rows; i += kFewWarps) {
            float top = -INFINITY, sum = 0.f, x[2][4] = {};
#pragma unroll
            for (int o = 0; o < kFewWarps; ++o) top = fmaxf(top, sh.m[o][i]);
#pragma unroll
            for (int o = 0; o < kFewWarps; ++o) {
                if (sh.m[o][i] == -INFINITY) {
                    sum += sh.l[o][i];                 // 0, or NaN where a visible score was
                    continue;
                }
                const float g = exp2_approx(sh.m[o][i] - top);
                sum = fmaf(g, sh.l[o][i], sum);
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (4 * lane + 128 * k < dv) {
                        float y[4];
                        load4(ring + o * kFewKeys * (kpitch + dv) + i * dv + 4 * lane + 128 * k, y);
#pragma unroll
                        for (int q = 0; q < 4; ++q) x[k][q] = fmaf(g, y[q], x[k][q]);
                    }
            }
            if (whole) {
                finish_row<float>(p, w, row0 + i, x, sum);
                continue;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (4 * lane + 128 * k < dv) store4(p.part + ((long long)slot * R + i) * dv + 4 * lane + 128 * k, x[k]);
            if (lane == 0) *(float2*)(p.ml + ((long long)slot * R + i) * 2) = make_float2(top, sum);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                   // the places are loaded into again
        __syncthreads();
    }
    if (!ok) *(volatile int*)p.error_flag = 1;
}

// ---- CUDA cores, more rows -----------------------------------------------------------------------------------------
// Tiles of 32 rows over blocks of 48 keys.  What bounds it next to multiply-adds is what shared memory can hand to the registers, 128 bytes a
// cycle, so a thread multiplies eight rows by six keys (eight apart), fourteen loads of 8 bytes for 96 products, and the head is dealt out in
// pairs of elements to the four lanes that have the same forty-eight; they hand each other their sums, so that each is left with two rows.  Weights pass
// through shared memory to the second product, eight rows times every sixteenth pair of columns over half of the keys a thread.  A warp owns its
// eight rows; only keys and values need all of them to meet.  They have one place each: the next block's keys are on their way under the
// softmax and the second product of this one, its values under the next scores.  Rows of keys are shifted by one 16-byte piece against each other,
// which meets no bank twice.
// Chunks of 100 tokens of three sequences, 16 heads of 72 over 4, the last 300 of up to 777 positions: 35 us, 5 of them to the first scores, 5 for the cut
// items.  128 tokens of four sequences up to 1024, heads of 128: 88.  (When these took 38 and 96: blocks of 64 keys 44 and 92, of 32 keys 40 and 109,
// four rows by two keys a thread 42 and 116.)
constexpr int kBlockRows = 32, kBlockKeys = 48, kKeysEach = kBlockKeys / 8, kBlockThreads = 128, kWarpRows = 8, kWeightPitch = kBlockKeys + 4;

struct BlockShared {
    uint64_t k_full, v_full, q_full;
    int gave_up;
};

struct BlockShape {
    size_t smem;
    int pairs;                                         // of columns a thread
    BlockShape(const zkfp_paged_attention_args& a)
    {
        pairs = (a.dv + 31) / 32;
        pairs = pairs <= 2 ? 2 : pairs <= 4 ? pairs : 8;
        smem = plan_bytes(a.batch) + sizeof(float) * ((size_t)kBlockKeys * (a.d + 4 + a.dv) + (size_t)kBlockRows * a.d + kBlockRows * kWeightPitch) +
               sizeof(BlockShared);
    }
};

template <typename T, int PAIRS>
__global__ void __launch_bounds__(kBlockThreads, PAIRS <= 3 ? 3 : 2)
paged_block_kernel(const __grid_constant__ Paged p)
{
    extern __shared__ __align__(16) uint8_t sm[];
    const zkfp_paged_attention_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = a.d, dv = a.dv, kpitch = d + 4, batch = (int)a.batch;
    const Plan plan(sm, batch);
    float* K = (float*)(sm + (((size_t)(batch + 1) * 8 + (size_t)batch * 12 + 15) & ~(size_t)15));            // [key][kpitch]
    float* V = K + kBlockKeys * kpitch;                                                                        // [key][dv]; at the end [row][dv]
    float* Q = V + kBlockKeys * dv;                                                                            // [row][d]
    float* P = Q + kBlockRows * d;                                                                             // [row][key]
    BlockShared& sh = *(BlockShared*)(P + kBlockRows * kWeightPitch);
    constexpr bool kBulk = sizeof(T) == 4;             // lines of keys and values go to shared memory as they are
    if (tid == 0) {
        mbar_init(smem_u32(&sh.k_full), kBlockKeys);
        mbar_init(smem_u32(&sh.v_full), kBlockKeys);
        mbar_init(smem_u32(&sh.q_full), kBlockRows);
        sh.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_enter();                                     // barriers touch nobody else
    make_plan(p, plan);
    const long long units = plan.before[batch];
    const Share share(p, units);
    const int cta = blockIdx.x;
    if (tid == 0) no_cut(p, cta);
    if (cta >= share.ctas || units == 0) return;
    const long long u1 = share.begin(cta + 1);
    long long u = share.begin(cta);
    // scores: keys kg + 8 e, pairs sp, sp + 4, ... of the head; then rows r0 and r0 + 1 of the warp's.  Values: column pairs cl + 16 k, keys 8 i + 4 kh + 0 .. 3.
    const int kg = lane & 7, sp = lane >> 3, r0 = 4 * (sp & 1) + 2 * (sp >> 1), cl = lane & 15, kh = lane >> 4;
    const float scale = a.scale * 1.4426950408889634f;
    uint32_t phase = 0, q_phase = 0;
    bool ok = true;
    Walk w;
    for (w.locate(p, plan, u); u < u1; w.next(p, plan)) {
        const int taken = (int)min((long long)w.left(p), u1 - u), j_begin = w.begin(p), j_end = w.end(p, taken);
        const long long end = u + w.left(p);
        u += taken;
        if (j_begin == j_end) continue;
        const bool whole = j_begin == 0 && j_end == w.count;
        if (tid == 0 && j_begin == 0 && !whole) write_cut(p, cta, share, w, end);
        const int slot = 2 * cta + (j_begin == 0 ? 1 : 0), row0 = w.t * kBlockRows, rows = min(kBlockRows, w.n * p.group - row0);
        const T *kb = (const T*)a.k + w.kv * a.k_head, *vb = (const T*)a.v + w.kv * a.v_head;
        // A thread asks for one line of a block, keys or values; its page is looked up a block ahead, and looked at when it is needed.
        auto find = [&](int j) {
            const int k = (w.first + j) * kBlockKeys + tid;
            return tid < kBlockKeys && j < j_end && k < w.len ? a.table[w.b * a.table_ld + (k >> p.shift)] : 0;
        };
        auto request = [&](int j, int page, bool values) {
            const int k0 = (w.first + j) * kBlockKeys;
            const T* from = values ? vb : kb;
            const long long page_step = values ? a.v_page : a.k_page, line_step = values ? a.v_pos : a.k_pos;
            float* to = values ? V : K;
            const int size = values ? dv : d, pitch = values ? dv : kpitch;
            if (kBulk) {
                if (tid >= kBlockKeys) return;
                const int k = k0 + tid;
                const bool there = k < w.len && page >= 0 && page < a.pages;
                if (k < w.len && !there) *(volatile int*)(p.error_flag + 1) = 1;
                const uint32_t bar = values ? smem_u32(&sh.v_full) : smem_u32(&sh.k_full);
                if (there) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // zeros that the line held
                    mbar_expect_tx(bar, size * 4);
                    bulk_load(smem_u32(to + tid * pitch), from + page * page_step + (k & (a.page - 1)) * line_step, size * 4, bar);
                } else {
                    for (int c = 0; c < size; c += 4) *(float4*)(to + tid * pitch + c) = make_float4(0.f, 0.f, 0.f, 0.f);
                    mbar_arrive(bar);
                }
            } else {
                for (int i = tid; i < kBlockKeys * (size / 4); i += kBlockThreads) {
                    const int n = i / (size / 4), c = 4 * (i - n * (size / 4)), k = k0 + n;
                    const long long at = k < w.len ? page_of(p, w.b, k) : -1;
                    if (k < w.len && at < 0) *(volatile int*)(p.error_flag + 1) = 1;
                    float x[4] = {};
                    if (at >= 0) load4(from + at * page_step + (k & (a.page - 1)) * line_step + c, x);
                    store4(to + n * pitch + c, x);
                }
            }
        };
        const int here = kBulk ? find(j_begin) : 0;
        int ahead = kBulk ? find(j_begin + 1) : 0;
        if (kBulk) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();                               // the item in front is done with all of it
        if (kBulk) {
            // rows behind the last hold what they held, and nothing reads their results
            if (tid >= kBlockThreads - kBlockRows) {
                const int n = tid - (kBlockThreads - kBlockRows), t = by_group(p, row0 + n), h = w.kv * p.group + row0 + n - t * p.group;
                mbar_expect_tx(smem_u32(&sh.q_full), n < rows ? d * 4 : 0);
                if (n < rows) bulk_load(smem_u32(Q + n * d), (const T*)a.q + (long long)(w.row0 + t) * a.q_tok + h * a.q_head, d * 4, smem_u32(&sh.q_full));
            }
        } else {
            for (int i = tid; i < rows * (d / 4); i += kBlockThreads) {
                const int n = i / (d / 4), c = (i - n * (d / 4)) * 4, t = by_group(p, row0 + n), h = w.kv * p.group + row0 + n - t * p.group;
                float x[4];
                load4((const T*)a.q + (long long)(w.row0 + t) * a.q_tok + h * a.q_head + c, x);
                store4(Q + n * d + c, x);
            }
        }
        request(j_begin, here, false);
        request(j_begin, here, true);
        if (kBulk) {
            if (ok) ok = mbar_wait_warp(smem_u32(&sh.q_full), q_phase, &sh.gave_up);
            q_phase ^= 1u;
        } else {
            __syncthreads();
        }
        const int row = kWarpRows * warp;              // the first of this warp's
        int pos[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) pos[i] = row + r0 + i < rows ? w.len - w.n + by_group(p, row0 + row + r0 + i) : -1;
        const int all_lo = first_seen(p, pos[1]);
        int column[PAIRS];                             // behind the last one: that one again, without a branch, and not stored
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) column[k] = min(32 * k + 2 * cl, dv - 2);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {};
        uint64_t acc[kWarpRows][PAIRS];
#pragma unroll
        for (int i = 0; i < kWarpRows; ++i)
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) acc[i][k] = 0;
        for (int j = j_begin; j < j_end; ++j) {
            const int k0 = (w.first + j) * kBlockKeys;
            const bool works = row < rows;             // this warp
            float s[kWarpRows][kKeysEach] = {};
            if (kBulk && ok) ok = mbar_wait_warp(smem_u32(&sh.k_full), phase, &sh.gave_up);
            if (works)
#pragma unroll 1
                for (int c = 2 * sp; c < d; c += 8) {
                    float2 q[kWarpRows];
#pragma unroll
                    for (int i = 0; i < kWarpRows; ++i) q[i] = *(const float2*)(Q + (row + i) * d + c);
#pragma unroll
                    for (int e = 0; e < kKeysEach; ++e) {
                        const float2 k = *(const float2*)(K + (kg + 8 * e) * kpitch + c);
#pragma unroll
                        for (int i = 0; i < kWarpRows; ++i) s[i][e] = fmaf(q[i].y, k.y, fmaf(q[i].x, k.x, s[i][e]));
                    }
                }
            __syncthreads();                           // the keys have been read
            if (j + 1 < j_end) request(j + 1, ahead, false);
            if (works) {
                // two of the eight rows, the four lanes' sums of them
                float h[4][kKeysEach], v[2][kKeysEach];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < kKeysEach; ++e) h[i][e] = (sp & 1 ? s[i + 4][e] : s[i][e]) + __shfl_xor_sync(0xffffffffu, sp & 1 ? s[i][e] : s[i + 4][e], 8);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < kKeysEach; ++e) v[i][e] = (sp & 2 ? h[i + 2][e] : h[i][e]) + __shfl_xor_sync(0xffffffffu, sp & 2 ? h[i][e] : h[i + 2][e], 16);
                const bool edge = pos[1] < 0 || k0 + kBlockKeys - 1 > pos[0] || k0 < all_lo;
                float top[2], f[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < kKeysEach; ++e) {
                        const int key = k0 + kg + 8 * e;
                        v[i][e] = edge && !(key <= pos[i] && (a.window <= 0 || pos[i] - key < a.window)) ? -INFINITY : v[i][e] * scale;
                        top[i] = e ? fmaxf(top[i], v[i][e]) : v[i][e];
                    }
#pragma unroll
                for (int o = 1; o < 8; o <<= 1)
#pragma unroll
                    for (int i = 0; i < 2; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    top[i] = fmaxf(top[i], m[i]);
                    const float sub = top[i] == -INFINITY ? 0.f : top[i];
                    f[i] = exp2_approx(m[i] - sub);
                    m[i] = top[i];
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < kKeysEach; ++e) {
                        v[i][e] = exp2_approx(v[i][e] - sub);
                        sum += v[i][e];
                        P[(row + r0 + i) * kWeightPitch + kg + 8 * e] = v[i][e];
                    }
                    l[i] = l[i] * f[i] + sum;          // of this lane's keys
                }
                if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                    for (int i = 0; i < kWarpRows; ++i) {
                        const uint64_t f2 = twice(__shfl_sync(0xffffffffu, f[i & 1], (i >> 2 & 1) * 8 + (i >> 1 & 1) * 16));
#pragma unroll
                        for (int k = 0; k < PAIRS; ++k) {
                            uint64_t y = 0;
                            fma2(y, acc[i][k], f2);
                            acc[i][k] = y;
                        }
                    }
                }
                __syncwarp();
            }
            if (kBulk && ok) ok = mbar_wait_warp(smem_u32(&sh.v_full), phase, &sh.gave_up);
            phase ^= 1u;
            if (works)
#pragma unroll 1
                for (int key = 4 * kh; key < kBlockKeys; key += 8) {
                    float x[kWarpRows][4];
#pragma unroll
                    for (int i = 0; i < kWarpRows; ++i) load4(P + (row + i) * kWeightPitch + key, x[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int k = 0; k < PAIRS; ++k) {
                            const uint64_t y = *(const uint64_t*)(V + (key + e) * dv + column[k]);
#pragma unroll
                            for (int i = 0; i < kWarpRows; ++i) fma2(acc[i][k], y, twice(x[i][e]));
                        }
                }
            __syncthreads();                           // the values have been read
            if (j + 1 < j_end) {
                request(j + 1, ahead, true);
                if (kBulk) ahead = find(j + 2);
            }
        }
        // both halves of the keys; the place of the values takes the rows of an item that is whole
        float* to = whole ? V : p.part + (long long)slot * p.tile * dv;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
            if (kg == 0 && row + r0 + i < rows) {
                if (whole) P[row + r0 + i] = l[i];
                else *(float2*)(p.ml + ((long long)slot * p.tile + row + r0 + i) * 2) = make_float2(m[i], l[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kWarpRows; ++i)
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                const uint64_t y = __shfl_xor_sync(0xffffffffu, acc[i][k], 16);
                const float x0 = __uint_as_float((uint32_t)acc[i][k]) + __uint_as_float((uint32_t)y);
                const float x1 = __uint_as_float((uint32_t)(acc[i][k] >> 32)) + __uint_as_float((uint32_t)(y >> 32));
                if (kh == (i & 1) && row + i < rows && 32 * k + 2 * cl < dv) *(float2*)(to + (row + i) * dv + 32 * k + 2 * cl) = make_float2(x0, x1);
            }
        if (whole) {
            __syncwarp();
            for (int i = row; i < min(row + kWarpRows, rows); ++i) {
                float x[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (4 * lane + 128 * k < dv) load4(V + i * dv + 4 * lane + 128 * k, x[k]);
                finish_row<T>(p, w, row0 + i, x, P[i]);
            }
        }
    }
    if (!ok) *(volatile int*)p.error_flag = 1;
}

// ---- cut items ---------------------------------------------------------------------------------------------------
// Block x merges the item that CTA x began and did not end, a warp per row.  Maxima are in units of log2 where base2.  Lanes take the
// parts' maxima and sums, 32 at a time, then all of them the columns of four parts at a time (eight: a prompt of 4096 173 instead of 169 us).
// Of large tiles a warp takes several rows, the next one's maxima and first two parts on their way under the one at work: blocks cost as
// much as the rows do (chunks of 100, 40 and 33 tokens with a block per four rows 24.3, 24.3 and 26.9 us, with 24 blocks 20.1, 18.4 and 25.0, with 12
// 22.8, 18.4 and 30.0).
constexpr int kMergeBlocks = 24;                       // per item of a large tile

template <typename T, int K, bool LARGE>
__global__ void __launch_bounds__(128)
paged_combine_kernel(const __grid_constant__ Paged p, int base2)
{
    chain_enter();
    const int c = blockIdx.x, lane = threadIdx.x & 31, dv = p.a.dv;
    const int4 what = *(const int4*)(p.cut + c * 8), where = *(const int4*)(p.cut + c * 8 + 4);
    const int parts = what.x;
    if (parts == 0) return;
    Walk w;
    w.b = what.y; w.kv = what.z; w.t = what.w;
    w.row0 = where.x; w.n = where.y; w.len = where.z;
    const int row0 = w.t * p.tile, rows = min(p.tile, w.n * p.group - row0);
    int r = blockIdx.y * 4 + (threadIdx.x >> 5);
    if (r >= rows) return;
    // the first part lies in the second place of its CTA, the others in the first of theirs
    auto place = [&](int i, int row) { return (2ll * (c + i) + (i == 0)) * p.tile + row; };
    auto maxima = [&](int i0, int row) {
        return i0 + lane < parts ? *(const float2*)(p.ml + place(i0 + lane, row) * 2) : make_float2(-INFINITY, 0.f);
    };
    auto columns = [&](int i, int row, float (&y)[K][4]) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (4 * lane + 128 * k < dv) load4(p.part + place(i, row) * dv + 4 * lane + 128 * k, y[k]);
    };
    constexpr int kAhead = LARGE ? 2 : 0;
    float2 ml = maxima(0, r);
    float ahead[2][K][4] = {};
#pragma unroll
    for (int e = 0; e < kAhead; ++e)
        if (e < parts) columns(e, r, ahead[e]);
    for (;;) {
        float x[K][4] = {}, m = -INFINITY, l = 0.f;
        const int next = r + 4 * gridDim.y;
        for (int i0 = 0; i0 < parts; i0 += 32) {
            const int n = min(parts - i0, 32);
            if (i0) ml = maxima(i0, r);
            const float m_new = fmaxf(m, warp_max(ml.x)), m_sub = m_new == -INFINITY ? 0.f : m_new;
            // A part without a score above -infinity has no say, whatever its sums are; its sum of weights is 0, or NaN where a visible score was,
            // which makes the row NaN and has it taken again.
            const float f = ml.x == -INFINITY ? 0.f : base2 ? exp2f(ml.x - m_sub) : expf(ml.x - m_sub);
            const float old = m == -INFINITY ? 0.f : base2 ? exp2f(m - m_sub) : expf(m - m_sub);
            l = l * old + (ml.x == -INFINITY ? ml.y : f * ml.y);
            m = m_new;
            const unsigned some = __ballot_sync(0xffffffffu, ml.x != -INFINITY);
            if (i0)
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int q = 0; q < 4; ++q) x[k][q] *= old;
            else {
#pragma unroll
                for (int e = 0; e < kAhead; ++e) {
                    const float g = __shfl_sync(0xffffffffu, f, e);
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int q = 0; q < 4; ++q) x[k][q] = some >> e & 1 ? fmaf(g, ahead[e][k][q], x[k][q]) : x[k][q];
                }
                if (LARGE && next < rows) {
                    if (parts <= 32) ml = maxima(0, next);
#pragma unroll
                    for (int e = 0; e < kAhead; ++e)
                        if (e < parts) columns(e, next, ahead[e]);
                }
            }
            for (int i = i0 ? 0 : kAhead; i < n; i += 4) {
                float y[4][K][4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        if (i + e < n && (some >> (i + e) & 1) && 4 * lane + 128 * k < dv) load4(p.part + place(i0 + i + e, r) * dv + 4 * lane + 128 * k, y[e][k]);
                        else y[e][k][0] = y[e][k][1] = y[e][k][2] = y[e][k][3] = 0.f;
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float g = __shfl_sync(0xffffffffu, f, (i + e) & 31);
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int q = 0; q < 4; ++q) x[k][q] = fmaf(g, y[e][k][q], x[k][q]);
                }
            }
        }
        finish_row<T>(p, w, row0 + r, x, warp_sum(l));
        if (!LARGE || (r = next) >= rows) return;
        if (parts > 32) ml = maxima(0, r);
    }
}

// ---- host --------------------------------------------------------------------------------------------------------
// CTAs that fit the GPU at once, `most` per SM
int grid_of(size_t smem, int most)
{
    const int per_sm = (int)(220 * 1024 / smem);
    return fp_sm_count() * (per_sm < 1 ? 1 : per_sm > most ? most : per_sm);
}

template <typename T>
int launch_combine(const Paged& p, int base2, cudaStream_t st)
{
    const long long bound = p.a.max_tokens * p.group < p.tile ? p.a.max_tokens * p.group : p.tile, most = (bound + 3) / 4;
    if (p.tile > 4 * kMergeBlocks) {
        const dim3 grid((unsigned)p.grid, (unsigned)(most < 1 ? 1 : most > kMergeBlocks ? kMergeBlocks : most));
        fp_launch(paged_combine_kernel<T, 1, true>, grid, dim3(128), 0, st, p, base2);          // dv <= 128
        return fp_launched();
    }
    const dim3 grid((unsigned)p.grid, (unsigned)(p.tile + 3) / 4);
    if (p.a.dv <= 128) fp_launch(paged_combine_kernel<T, 1, false>, grid, dim3(128), 0, st, p, base2);
    else fp_launch(paged_combine_kernel<T, 2, false>, grid, dim3(128), 0, st, p, base2);
    return fp_launched();
}

int launch_plain(Paged& p, cudaStream_t st)
{
    const PlainShape<bf16> s(p.a);
    if (s.smem > (size_t)kSharedMax) return ZKDS_ERR_UNSUPPORTED;
    ZKDS_CUDA(cudaFuncSetAttribute(paged_plain_kernel<bf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    fp_launch(paged_plain_kernel<bf16>, dim3((unsigned)p.grid), dim3(kPlainThreads), s.smem, st, p, s.kpitch);
    const int rc = fp_launched();
    return rc != ZKDS_OK ? rc : launch_combine<bf16>(p, 0, st);
}

template <int R, int PAIRS>
int launch_few(Paged& p, cudaStream_t st)
{
    const size_t smem = few_bytes<R>(p.a);
    if (smem > (size_t)kSharedMax) return ZKDS_ERR_UNSUPPORTED;
    ZKDS_CUDA(cudaFuncSetAttribute(paged_few_kernel<R, PAIRS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    fp_launch(paged_few_kernel<R, PAIRS>, dim3((unsigned)p.grid), dim3(kFewThreads), smem, st, p);
    const int rc = fp_launched();
    return rc != ZKDS_OK ? rc : launch_combine<float>(p, 1, st);
}

template <int R>
int launch_few(Paged& p, cudaStream_t st)
{
    return p.a.dv <= 64 ? launch_few<R, 2>(p, st) : p.a.dv <= 128 ? launch_few<R, 4>(p, st) : launch_few<R, 8>(p, st);
}

template <typename T, int PAIRS>
int launch_block(Paged& p, size_t smem, cudaStream_t st)
{
    ZKDS_CUDA(cudaFuncSetAttribute(paged_block_kernel<T, PAIRS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    fp_launch(paged_block_kernel<T, PAIRS>, dim3((unsigned)p.grid), dim3(kBlockThreads), smem, st, p);
    const int rc = fp_launched();
    return rc != ZKDS_OK ? rc : launch_combine<T>(p, 1, st);
}

template <typename T>
int launch_cores(Paged& p, cudaStream_t st)
{
    if (p.tile == 4) return launch_few<4>(p, st);
    if (p.tile == 8) return launch_few<8>(p, st);
    if (p.tile == kPlainRows) return launch_plain(p, st);
    const BlockShape s(p.a);
    if (s.smem > (size_t)kSharedMax) return ZKDS_ERR_UNSUPPORTED;
    switch (s.pairs) {
    case 2: return launch_block<T, 2>(p, s.smem, st);
    case 3: return launch_block<T, 3>(p, s.smem, st);
    case 4: return launch_block<T, 4>(p, s.smem, st);
    default: return launch_block<T, 8>(p, s.smem, st);
    }
}

// grid and tile of the kernel that a call takes
void choose_kernel(Paged& p)
{
    const int path = zkfp_paged_path(&p.a);
    if (path == 2) return paged_stream_shape(p);
    if (path == 1) return paged_tile_shape(p);
    const long long rows = p.a.max_tokens * p.group;
    p.over = 1;
    p.least = 1;
    if (p.a.dtype != ZKFP_BF16 && rows <= kFewRows) {
        p.tile = rows <= 4 ? 4 : 8;
        p.block = kFewBlock;
        p.over = 2;
        p.grid = grid_of(rows <= 4 ? few_bytes<4>(p.a) : few_bytes<8>(p.a), p.a.dv <= 128 ? 3 : 2);
    } else if (rows <= kPlainRows) {
        p.tile = kPlainRows;
        p.block = kPlainKeys;
        p.grid = grid_of(PlainShape<bf16>(p.a).smem, 6);
    } else {
        const BlockShape s(p.a);
        p.tile = kBlockRows;
        p.block = kBlockKeys;
        p.grid = grid_of(s.smem, s.pairs <= 3 ? 3 : 2);
    }
}

// (so that products with it stay in range)
void bound_tokens(zkfp_paged_attention_args& a)
{
    if (a.max_tokens > 1 << 30) a.max_tokens = 1 << 30;
}

void choose(Paged& p)
{
    bound_tokens(p.a);
    p.shift = page_shift(p.a.page);
    p.group = p.a.heads / p.a.kv_heads;
    choose_kernel(p);
    p.by_groups.set(p.group);
    p.by_tiles.set(p.tile);
    p.by_blocks.set(p.block);
    p.by_heads.set(p.a.kv_heads);
}

bool paged_ok(const zkfp_paged_attention_args* a)
{
    return a && a->q && a->k && a->v && a->out && a->table && a->rows && a->lengths && a->tokens >= 0 && a->pages > 0 && a->table_cols > 0 &&
           a->table_ld >= a->table_cols && a->batch > 0 && a->max_tokens >= 0 && a->kv_heads > 0 && a->heads > 0 &&
           a->heads % a->kv_heads == 0 && a->scale >= 0.f && a->scale < 3e38f && a->window >= 0 && !((uintptr_t)a->scratch & 31) && a->d > 0 && a->dv > 0 && !(a->d & 7) && !(a->dv & 7) && page_shift(a->page) >= 0 && (unsigned)a->dtype <= 1 &&
           !((a->q_tok | a->q_head | a->k_page | a->k_pos | a->k_head | a->v_page | a->v_pos | a->v_head | a->o_tok | a->o_head | a->gate_tok |
              a->gate_head) & 7) &&
           !(((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out | (uintptr_t)a->gate) & 15);
}

bool paged_takes(const zkfp_paged_attention_args* a)
{
    return a->batch <= kPagedBatch && a->d <= kPlainMost && a->dv <= kPlainMost && a->tokens < 0x40000000ll / a->heads && a->pages <= 0x7fffffffll;
}

}  // namespace

}  // namespace zkds

using namespace zkds;

extern "C" {

int zkfp_paged_path(const zkfp_paged_attention_args* a)
{
    if (!a || a->heads <= 0 || a->kv_heads <= 0 || a->heads < a->kv_heads || a->d <= 0 || a->dv <= 0 || a->batch <= 0) return 0;
    zkfp_paged_attention_args b = *a;
    bound_tokens(b);
    if (paged_stream_takes(b)) return 2;
    return paged_tile_takes(b) ? 1 : 0;
}

long long zkfp_paged_scratch(const zkfp_paged_attention_args* a)
{
    if (!paged_ok(a) || !paged_takes(a)) return 0;
    Paged p;
    p.a = *a;
    choose(p);
    return 2ll * p.grid * p.tile * (a->dv + 2) + 8ll * p.grid;
}

int zkfp_paged_attention(const zkfp_paged_attention_args* a, void* stream)
{
    if (!paged_ok(a)) return ZKDS_ERR_ARG;
    if (!paged_takes(a)) return ZKDS_ERR_UNSUPPORTED;
    if (a->tokens == 0) return ZKDS_OK;
    if (!a->scratch) return ZKDS_ERR_ARG;
    Paged p;
    p.a = *a;
    choose(p);
    p.part = a->scratch;
    p.ml = a->scratch + 2ll * p.grid * p.tile * a->dv;
    p.cut = (int*)(p.ml + 4ll * p.grid * p.tile);
    p.error_flag = fp_error_flag();
    if (!p.error_flag) return ZKDS_ERR_WORKSPACE;
    cudaStream_t st = (cudaStream_t)stream;
    const int path = zkfp_paged_path(a);
    if (path) {
        const int rc = path == 2 ? launch_paged_stream(p, st) : launch_paged_tile(p, st);
        return rc != ZKDS_OK ? rc : launch_combine<bf16>(p, 1, st);
    }
    return a->dtype == ZKFP_BF16 ? launch_cores<bf16>(p, st) : launch_cores<float>(p, st);
}

}  // extern "C"
