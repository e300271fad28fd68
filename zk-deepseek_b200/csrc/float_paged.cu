// Attention of new tokens over pages: the kernels of CUDA cores (float32, and sizes that the tensor cores do not take) and
// the one that merges what the CTAs of a cut item leave.  How the work is shared is in float_paged.cuh.
#include "float_paged.cuh"

namespace zkds {

namespace {

// ---- CUDA cores, few rows ----------------------------------------------------------------------------------------
// Tiles of 16 rows over blocks of 64 keys, all in shared memory, sums of a row in registers: a thread holds eight columns of
// up to four rows.
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
    const int ctas = sharing(p, units), cta = blockIdx.x;
    if (tid == 0) no_cut(p, cta);
    if (cta >= ctas || units == 0) return;
    const long long u1 = range_begin(units, cta + 1, ctas);
    long long u = range_begin(units, cta, ctas);
    Walk w;
    for (w.locate(p, plan, u); u < u1; w.next(p, plan)) {
        const int taken = (int)min((long long)w.left(p), u1 - u), j_begin = w.begin(p), j_end = w.end(p, taken);
        const long long end = u + w.left(p);
        u += taken;
        if (j_begin == j_end) continue;
        const bool whole = j_begin == 0 && j_end == w.count;
        if (tid == 0 && j_begin == 0 && !whole) write_cut(p, cta, units, ctas, w, end);
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
                if (r < nk && page < 0) *(volatile int*)p.error_flag = 1;
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

// ---- CUDA cores, more rows -----------------------------------------------------------------------------------------
// Tiles of 32 rows over blocks of 64 keys, which bound it by multiply-adds: sixteen lanes own four rows.  Scores: four rows times four keys (16
// apart) a thread, two products an instruction along the head, so that eight 16-byte loads feed 64 products; rows of keys are shifted by one
// 16-byte piece against each other, which meets no bank twice.  The rows' maxima and sums are these lanes' own, and so are the weights, which pass through shared memory to the second product: four rows times every
// sixteenth pair of columns.  Only the keys and values need the whole block to meet.
constexpr int kBlockRows = 32, kBlockKeys = 64, kBlockThreads = 128, kWeightPitch = kBlockKeys + 4;

struct BlockShape {
    size_t smem;
    int pairs;                                         // of columns a thread
    BlockShape(const zkfp_paged_attention_args& a)
    {
        pairs = (a.dv + 31) / 32;
        pairs = pairs <= 2 ? 2 : pairs <= 4 ? pairs : 8;
        smem = plan_bytes(a.batch) + sizeof(float) * ((size_t)kBlockKeys * (a.d + 4 + a.dv) + (size_t)kBlockRows * a.d + kBlockRows * kWeightPitch);
    }
};

template <typename T, int PAIRS>
__global__ void __launch_bounds__(kBlockThreads)
paged_block_kernel(const __grid_constant__ Paged p)
{
    chain_enter();
    extern __shared__ __align__(16) uint8_t sm[];
    const zkfp_paged_attention_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, d = a.d, dv = a.dv, vd = d / 8, pieces = vd + dv / 8, kpitch = d + 4, batch = (int)a.batch;
    const Plan plan(sm, batch);
    float* K = (float*)(sm + (((size_t)(batch + 1) * 8 + (size_t)batch * 12 + 15) & ~(size_t)15));            // [key][kpitch]
    float* Q = K + kBlockKeys * kpitch;                                                                        // [row][d]
    float* V = Q + kBlockRows * d;                                                                             // [key][dv]; at the end [row][dv]
    float* P = V + kBlockKeys * dv;                                                                            // [row][key]
    make_plan(p, plan);
    const long long units = plan.before[batch];
    const int ctas = sharing(p, units), cta = blockIdx.x;
    if (tid == 0) no_cut(p, cta);
    if (cta >= ctas || units == 0) return;
    const long long u1 = range_begin(units, cta + 1, ctas);
    long long u = range_begin(units, cta, ctas);
    const int r4 = tid >> 4, at = tid & 15;            // which four rows, which of the sixteen
    Walk w;
    for (w.locate(p, plan, u); u < u1; w.next(p, plan)) {
        const int taken = (int)min((long long)w.left(p), u1 - u), j_begin = w.begin(p), j_end = w.end(p, taken);
        const long long end = u + w.left(p);
        u += taken;
        if (j_begin == j_end) continue;
        const bool whole = j_begin == 0 && j_end == w.count;
        if (tid == 0 && j_begin == 0 && !whole) write_cut(p, cta, units, ctas, w, end);
        const int slot = 2 * cta + (j_begin == 0 ? 1 : 0), row0 = w.t * kBlockRows, rows = min(kBlockRows, w.n * p.group - row0);
        __syncthreads();
        for (int i = tid; i < kBlockRows * vd; i += kBlockThreads) {
            const int r = i / vd, c = (i - r * vd) * 8;
            float x[8] = {};
            if (r < rows) {
                const int t = by_group(p, row0 + r), h = w.kv * p.group + row0 + r - t * p.group;
                load8((const T*)a.q + (long long)(w.row0 + t) * a.q_tok + h * a.q_head + c, x);
            }
            store8(Q + r * d + c, x);
        }
        int pos[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pos[i] = 4 * r4 + i < rows ? w.len - w.n + by_group(p, row0 + 4 * r4 + i) : -1;
        int column[PAIRS];                             // behind the last one: that one again, without a branch, and not stored
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) column[k] = min(32 * k + 2 * at, dv - 2);
        float m[4], l[4];
        uint64_t acc[4][PAIRS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) acc[i][k] = 0;
        }
        for (int j = j_begin; j < j_end; ++j) {
            const int k0 = (w.first + j) * kBlockKeys;
            __syncthreads();                           // the block in front is done with keys and values
            {
                // a warp takes every fourth key with its value, a lane a piece; lane i knows the page of the i-th
                const int warp = tid >> 5, of = k0 + warp + 4 * (lane & 15);
                const long long held = of < w.len ? page_of(p, w.b, of) : -1;
                if (of < w.len && held < 0) *(volatile int*)p.error_flag = 1;
                __syncwarp();
                for (int c = lane; c < (pieces + 31) / 32 * 32; c += 32) {
                    const bool key = c < vd;
                    const T* base = key ? (const T*)a.k + w.kv * a.k_head + 8 * c : (const T*)a.v + w.kv * a.v_head + 8 * (c - vd);
                    const long long page_step = key ? a.k_page : a.v_page, line_step = key ? a.k_pos : a.v_pos;
                    float* to = key ? K + 8 * c : V + 8 * (c - vd);
                    const int to_step = key ? kpitch : dv;
#pragma unroll 8
                    for (int i = 0; i < kBlockKeys / 4; ++i) {
                        const int r = warp + 4 * i;
                        const long long page = __shfl_sync(0xffffffffu, held, i);
                        float x[8] = {};
                        if (page >= 0 && c < pieces) load8(base + page * page_step + ((k0 + r) & (a.page - 1)) * line_step, x);
                        if (c < pieces) store8(to + r * to_step, x);
                    }
                }
            }
            __syncthreads();
            if (4 * r4 >= rows) continue;              // sixteen lanes without rows
            uint64_t s[4][4] = {};                     // even and odd elements apart
#pragma unroll 2
            for (int c = 0; c < d; c += 4) {
                ulonglong2 q[4], k[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    q[i] = *(const ulonglong2*)(Q + (4 * r4 + i) * d + c);
                    k[i] = *(const ulonglong2*)(K + (at + 16 * i) * kpitch + c);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        fma2(s[i][e], q[i].x, k[e].x);
                        fma2(s[i][e], q[i].y, k[e].y);
                    }
            }
            const unsigned half = 0xffffu << (lane & 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4], top = m[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = k0 + at + 16 * e;
                    const bool seen = key <= pos[i] && (a.window <= 0 || pos[i] - key < a.window);
                    v[e] = seen ? (__uint_as_float((uint32_t)s[i][e]) + __uint_as_float((uint32_t)(s[i][e] >> 32))) * a.scale : -INFINITY;
                    top = fmaxf(top, v[e]);
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(half, top, o));
                const float f = m[i] == -INFINITY ? 0.f : expf(m[i] - top);
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = v[e] == -INFINITY ? 0.f : expf(v[e] - top);
                    sum += v[e];
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(half, sum, o);
                l[i] = l[i] * f + sum;
                m[i] = top;
                const uint64_t f2 = twice(f);
                uint64_t none = 0;
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) {
                    uint64_t y = none;
                    fma2(y, acc[i][k], f2);
                    acc[i][k] = y;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) P[(4 * r4 + i) * kWeightPitch + at + 16 * e] = v[e];
            }
            __syncwarp(half);
            for (int key = 0; key < kBlockKeys; key += 4) {
                float x[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) load4(P + (4 * r4 + i) * kWeightPitch + key, x[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) {
                        const uint64_t v = *(const uint64_t*)(V + (key + e) * dv + column[k]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) fma2(acc[i][k], v, twice(x[i][e]));
                    }
            }
        }
        __syncthreads();                               // the values make room for the sums
        float* to = whole ? V : p.part + (long long)slot * p.tile * dv;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (4 * r4 + i >= rows) break;
#pragma unroll
            for (int k = 0; k < PAIRS; ++k)
                if (32 * k + 2 * at < dv) *(uint64_t*)(to + (4 * r4 + i) * dv + 32 * k + 2 * at) = acc[i][k];
            if (at == 0) {
                if (whole) P[4 * r4 + i] = l[i];
                else *(float2*)(p.ml + ((long long)slot * p.tile + 4 * r4 + i) * 2) = make_float2(m[i], l[i]);
            }
        }
        if (whole) {
            __syncthreads();
            for (int r = tid >> 5; r < rows; r += kBlockThreads / 32) {
                float x[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (4 * lane + 128 * k < dv) load4(V + r * dv + 4 * lane + 128 * k, x[k]);
                finish_row<T>(p, w, row0 + r, x, P[r]);
            }
        }
    }
}

// ---- cut items ---------------------------------------------------------------------------------------------------
// Block x merges the item that CTA x began and did not end, a warp per row.  Maxima are in units of log2 where base2.  Lanes take the
// parts' maxima and sums, 32 at a time, then all of them the columns of eight parts at a time.
template <typename T, int K>
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
    const int r = blockIdx.y * 4 + (threadIdx.x >> 5);
    if (r >= rows) return;
    // the first part lies in the second place of its CTA, the others in the first of theirs
    auto place = [&](int i) { return (2ll * (c + i) + (i == 0)) * p.tile + r; };
    float x[K][4] = {}, m = -INFINITY, l = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 32) {
        const int n = min(parts - i0, 32);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < n) ml = *(const float2*)(p.ml + place(i0 + lane) * 2);
        const float m_new = fmaxf(m, warp_max(ml.x)), m_sub = m_new == -INFINITY ? 0.f : m_new;
        // a part without a key that the row sees has no say, whatever its sums are
        const float f = ml.x == -INFINITY ? 0.f : base2 ? exp2f(ml.x - m_sub) : expf(ml.x - m_sub);
        const float old = m == -INFINITY ? 0.f : base2 ? exp2f(m - m_sub) : expf(m - m_sub);
        l = l * old + (ml.x == -INFINITY ? 0.f : f * ml.y);
        m = m_new;
        const unsigned some = __ballot_sync(0xffffffffu, ml.x != -INFINITY);
        if (i0)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q) x[k][q] *= old;
        for (int i = 0; i < n; i += 8) {
            float y[8][K][4];
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (i + e < n && (some >> (i + e) & 1) && 4 * lane + 128 * k < dv) load4(p.part + place(i0 + i + e) * dv + 4 * lane + 128 * k, y[e][k]);
                    else y[e][k][0] = y[e][k][1] = y[e][k][2] = y[e][k][3] = 0.f;
                }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float g = __shfl_sync(0xffffffffu, f, (i + e) & 31);
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int q = 0; q < 4; ++q) x[k][q] = fmaf(g, y[e][k][q], x[k][q]);
            }
        }
    }
    finish_row<T>(p, w, row0 + r, x, warp_sum(l));
}

// ---- host --------------------------------------------------------------------------------------------------------
template <typename T>
int plain_grid(const zkfp_paged_attention_args& a)
{
    const size_t smem = PlainShape<T>(a).smem;
    const int per_sm = (int)(220 * 1024 / smem);
    return fp_sm_count() * (per_sm < 1 ? 1 : per_sm > 6 ? 6 : per_sm);
}

template <typename T>
int launch_combine(const Paged& p, int base2, cudaStream_t st)
{
    const dim3 grid((unsigned)p.grid, (unsigned)(p.tile + 3) / 4);
    if (p.a.dv <= 128) fp_launch(paged_combine_kernel<T, 1>, grid, dim3(128), 0, st, p, base2);
    else fp_launch(paged_combine_kernel<T, 2>, grid, dim3(128), 0, st, p, base2);
    return fp_launched();
}

template <typename T>
int launch_plain(Paged& p, cudaStream_t st)
{
    const PlainShape<T> s(p.a);
    if (s.smem > (size_t)kSharedMax) return ZKDS_ERR_UNSUPPORTED;
    ZKDS_CUDA(cudaFuncSetAttribute(paged_plain_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    fp_launch(paged_plain_kernel<T>, dim3((unsigned)p.grid), dim3(kPlainThreads), s.smem, st, p, s.kpitch);
    const int rc = fp_launched();
    return rc != ZKDS_OK ? rc : launch_combine<T>(p, 0, st);
}

template <typename T, int PAIRS>
int launch_block(Paged& p, size_t smem, cudaStream_t st)
{
    ZKDS_CUDA(cudaFuncSetAttribute(paged_block_kernel<T, PAIRS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    fp_launch(paged_block_kernel<T, PAIRS>, dim3((unsigned)p.grid), dim3(kBlockThreads), smem, st, p);
    const int rc = fp_launched();
    return rc != ZKDS_OK ? rc : launch_combine<T>(p, 0, st);
}

template <typename T>
int launch_cores(Paged& p, cudaStream_t st)
{
    if (p.tile == kPlainRows) return launch_plain<T>(p, st);
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
void choose(Paged& p)
{
    p.shift = page_shift(p.a.page);
    set_group(p, p.a.heads / p.a.kv_heads);
    const int path = zkfp_paged_path(&p.a);
    if (path == 2) return paged_stream_shape(p);
    if (path == 1) return paged_tile_shape(p);
    p.block = kPlainKeys;
    p.over = 1;
    p.least = 2;
    if (p.a.max_tokens * p.group > kPlainRows) {
        p.tile = kBlockRows;
        const int per_sm = (int)(220 * 1024 / BlockShape(p.a).smem);
        p.grid = fp_sm_count() * (per_sm < 1 ? 1 : per_sm > 4 ? 4 : per_sm);
        return;
    }
    p.tile = kPlainRows;
    p.grid = p.a.dtype == ZKFP_BF16 ? plain_grid<bf16>(p.a) : plain_grid<float>(p.a);
}

bool paged_ok(const zkfp_paged_attention_args* a)
{
    return a && a->q && a->k && a->v && a->out && a->table && a->rows && a->lengths && a->tokens >= 0 && a->pages > 0 && a->table_cols > 0 &&
           a->table_ld >= a->table_cols && a->batch > 0 && a->max_tokens >= 0 && a->kv_heads > 0 && a->heads > 0 &&
           a->heads % a->kv_heads == 0 && a->scale >= 0.f && a->scale < 3e38f && a->window >= 0 && !((uintptr_t)a->scratch & 15) && a->d > 0 && a->dv > 0 && !(a->d & 7) && !(a->dv & 7) && page_shift(a->page) >= 0 && (unsigned)a->dtype <= 1 &&
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
    if (paged_stream_takes(*a)) return 2;
    return paged_tile_takes(*a) ? 1 : 0;
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
