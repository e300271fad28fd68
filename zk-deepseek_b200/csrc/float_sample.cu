// One token per row of logits from given random numbers: temperature, the k largest, the likeliest p, at least min_p.
//
// Weights are w = 2^((l - max) log2(e) / temperature), held as whole multiples of 2^-44: their sums are exact in any order, so
// that neither the threads' timing nor the shape of the launch moves a border between two tokens.  2^y is made in 64 bits: y
// by one product, 2^y from a table of 2^(i / 256) and the series of 2^r, |r| <= 1 / 512, to its fourth power (the fifth is 2^-54).
//
// A row belongs to a cluster of 1 to 8 CTAs, each of which keeps its slice of the row in shared memory, so the row is read from memory
// once.  What a row keeps is a prefix of its tokens in falling order of rank: the logit, then the lower index.  The prefix's last token is found in two steps: a histogram of 1024 equal stretches
// between the smallest and the largest logit, of counts or of weights, names the stretch that it lies in; the tokens of that
// stretch, a few hundred at most on logits of a model, meet in the first CTA, which ranks them.  Where they are more than its list
// holds (logits that are equal, or nearly), the key is found 8 bits at a time instead.
//
// Latency bounds it: a pass over the row for each limit and one for the draw, and the cluster's barriers between them.  One row of 129280 with top p
// 20 to 27 us (8 without a limit), 64 rows of 32768 with top k 16, 256 rows of 129280 with limits of their own 191: 37 rows at a time, as many as
// shared memory holds, for reading a row again from memory for every pass costs more (265).
#include <cooperative_groups.h>

#include "float_common.cuh"

namespace zkds {

namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32, kStretches = 1024, kListed = 1024, kClusterMost = 8;

// what a logit counts as: NaN as -infinity, both zeros as one
__device__ __forceinline__ float plain_logit(float l) { return l != l ? -INFINITY : l + 0.f; }
// its bits in the order of whole numbers
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t u = __float_as_uint(l);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ uint64_t rank_of(float l, uint32_t index) { return (uint64_t)key_of(l) << 32 | (uint32_t)~index; }

struct Weigher {
    const double* table;             // 2^(i / 256)
    double top, scale;               // scale: 256 log2(e) / temperature
    float cut, most;                 // smaller logits weigh nothing, larger (infinite) ones are all alike
    // 256 times the exponent
    __device__ __forceinline__ double exponent(float l) const { return ((double)fminf(l, most) - top) * scale; }
    // without a branch, so that the chains of several logits run side by side
    __device__ __forceinline__ uint64_t operator()(float l) const
    {
        const double y = exponent(l);
        const double magic = 6755399441055744.0;       // 1.5 * 2^52: adding it rounds to a whole number, in the low bits
        const double n = y + magic, r = y - (n - magic), c = 0.0027076061740622863;              // ln(2) / 256
        const int i = __double2loint(n);
        const double t = table[i & 255], e = fma(r, fma(r, fma(r, fma(r, c * c * c * c / 24, c * c * c / 6), c * c / 2), c), 1.0);
        // times 2^44 and the whole part, in the exponent; adding 2^52 leaves the rounded number in the low bits
        const double w = e * __hiloint2double(__double2hiint(t) + ((i >> 8) + 44) * 0x100000, __double2loint(t)) + 4503599627370496.0;
        return l < cut ? 0 : (uint64_t)__double_as_longlong(w) & 0xfffffffffffffull;
    }
};

struct SampleShared {
    double table[256];
    unsigned long long hist[kStretches];               // weight, or number, of the tokens of a stretch
    unsigned long long list[kListed];                  // ranks of the border's tokens (first CTA)
    unsigned listed;
    unsigned count[256];
    float best[kClusterMost], least[kClusterMost];
    uint32_t first[kClusterMost];
    unsigned long long share[kClusterMost], share2[kClusterMost];
    unsigned long long found[2], border;               // stretch and what is in front of it; rank of the last token kept
    unsigned long long red[kSampleWarps], red2[kSampleWarps];
};

__device__ __forceinline__ uint64_t warp_scan64(uint64_t v)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
    }
    return v;
}
__device__ __forceinline__ uint64_t warp_add64(uint64_t v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// 64-bit sums in two words, each by a native atomic: a word that passes 2^32 hands its carry on
__device__ __forceinline__ void add_weight(unsigned long long* sum, uint64_t w)
{
    unsigned* word = (unsigned*)sum;
    const unsigned a = (unsigned)w, old = atomicAdd(word, a), up = (unsigned)(w >> 32) + (old + a < old ? 1u : 0u);
    if (up) atomicAdd(word + 1, up);
}

template <typename T, int C>
struct Sampler {
    cg::cluster_group cluster;
    SampleShared& s;
    const float* logits;                               // this CTA's, four at a time, -infinity behind the last
    int fours, base, me, tid, lane, warp;              // groups of four, index of the first
    Weigher weight;
    float top, per;                                    // stretches per logit
    float low;                                         // kept: logits above it, and those equal to it in front of this index
    uint32_t upto;

    __device__ __forceinline__ SampleShared& of(int r) { return C == 1 ? s : *cluster.map_shared_rank(&s, r); }
    __device__ __forceinline__ void sync()
    {
        if (C == 1) __syncthreads();
        else cluster.sync();
    }
    __device__ __forceinline__ bool kept(float l, uint32_t index) const { return l > low || (l == low && index < upto); }
    // which stretch a logit lies in, before rounding down
    __device__ __forceinline__ float place(float l) const { return (top - fminf(l, top)) * per; }
    __device__ __forceinline__ int stretch(float l) const { return (int)fminf(place(l), (float)(kStretches - 1)); }
    // f(i, four logits) of the groups of four that may hold some that are kept
    template <typename F>
    __device__ __forceinline__ void each(F f)
    {
        for (int i = tid; i < fours; i += kSampleThreads) {
            const float4 v = *reinterpret_cast<const float4*>(logits + 4 * i);
            if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) < low) continue;
            const float x[4] = {v.x, v.y, v.z, v.w};
            f(base + 4 * i, x);
        }
    }

    // (of a copy, so that the fields of the one at work stay in registers)
    static __device__ __noinline__ void by_bits(Sampler p, bool by_weight, double limit, int border, uint64_t before) { p.by_bits(by_weight, limit, border, before); }

    // the prefix of `wanted` tokens, or (by weight) up to the token in front of which lies a share of p of all weight or more
    __device__ __forceinline__ void narrow(bool by_weight, uint64_t wanted, double p)
    {
        __syncthreads();
        for (int i = tid; i < kStretches; i += kSampleThreads) s.hist[i] = 0;
        if (tid == 0) s.listed = 0;
        __syncthreads();
        if (by_weight)
            each([&](uint32_t index, const float (&x)[4]) {
                uint64_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = weight(x[k]);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (w[k] && kept(x[k], index + k)) add_weight(&s.hist[stretch(x[k])], w[k]);
            });
        else
            each([&](uint32_t index, const float (&x)[4]) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (kept(x[k], index + k)) atomicAdd((unsigned*)&s.hist[stretch(x[k])], 1u);
            });
        sync();
        // Every CTA sums its share of the stretches over all CTAs.  (Each summing all of them, which saves two barriers, takes longer: 5 us for
        // 64 KB from the shared memory of seven others.)
        constexpr int kMine = kStretches / C, kPer = (kMine + kSampleThreads - 1) / kSampleThreads;
        uint64_t v[kPer], mine = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            v[k] = 0;
            if (tid * kPer < kMine)
#pragma unroll
                for (int r = 0; r < C; ++r) v[k] += of(r).hist[me * kMine + tid * kPer + k];
            mine += v[k];
        }
        uint64_t run = warp_scan64(mine);
        if (lane == 31) s.red[warp] = run;
        __syncthreads();
        uint64_t sum = 0, before = run - mine, total = 0;
        for (int i = 0; i < kSampleWarps; ++i) {
            if (i < warp) before += s.red[i];
            sum += s.red[i];
        }
        if (tid < C) of(tid).share[me] = sum;
        sync();
        for (int r = 0; r < C; ++r) {
            if (r < me) before += s.share[r];
            total += s.share[r];
        }
        if (!by_weight && wanted >= total) return;                     // the same in every CTA
        const double limit = by_weight ? fmax(p * (double)total, 1.0) : (double)wanted;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (tid * kPer < kMine && (double)before < limit && (double)(before + v[k]) >= limit)
                for (int r = 0; r < C; ++r) {
                    of(r).found[0] = me * kMine + tid * kPer + k;
                    of(r).found[1] = before;
                }
            before += v[k];
        }
        sync();
        const int border = (int)s.found[0];
        before = s.found[1];
        SampleShared& one = of(0);
        const float first = (float)border, end = border == kStretches - 1 ? INFINITY : first + 1.0f;
        each([&](uint32_t index, const float (&x)[4]) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = place(x[k]);
                if (f < first || !(f < end || border == kStretches - 1) || !kept(x[k], index + k)) continue;
                const unsigned at = atomicAdd(&one.listed, 1u);
                if (at < kListed) one.list[at] = rank_of(x[k], index + k);
            }
        });
        sync();
        if (one.listed <= kListed) {
            if (me == 0) {
                const int m = (int)s.listed;
                unsigned long long* w = s.hist;
                for (int i = tid; i < m; i += kSampleThreads) w[i] = by_weight ? weight(logit_of((uint32_t)(s.list[i] >> 32))) : 1;
                __syncthreads();
                for (int i = tid; i < m; i += kSampleThreads) {
                    const uint64_t rank = s.list[i];
                    uint64_t in_front = before;
                    for (int k = 0; k < m; ++k) in_front += s.list[k] > rank ? w[k] : 0;
                    if ((double)in_front < limit && (double)(in_front + w[i]) >= limit)
                        for (int r = 0; r < C; ++r) of(r).border = rank;
                }
            }
        } else {
            by_bits(*this, by_weight, limit, border, before);
        }
        sync();
        low = logit_of((uint32_t)(s.border >> 32));
        upto = ~(uint32_t)s.border + 1;
    }

    // the same among the many tokens of one stretch
    __device__ __forceinline__ void by_bits(bool by_weight, double limit, int border, uint64_t before)
    {
        uint32_t prefix = 0;
        uint64_t here = 0;
        for (int bits = 24; bits >= 0; bits -= 8) {
            if (tid < 256) s.hist[tid] = s.count[tid] = 0;
            __syncthreads();
            each([&](uint32_t index, const float (&x)[4]) {
                for (int k = 0; k < 4; ++k) {
                    const uint32_t key = key_of(x[k]);
                    if (!kept(x[k], index + k) || stretch(x[k]) != border || (bits < 24 && key >> (bits + 8) != prefix >> (bits + 8))) continue;
                    const int d = (key >> bits) & 255;
                    atomicAdd(&s.count[d], 1u);
                    const uint64_t w = by_weight ? weight(x[k]) : 1;
                    if (w) add_weight(&s.hist[d], w);
                }
            });
            sync();
            // every CTA looks through the sums of all, from the largest digit down
            if (tid < 256) {
                uint64_t sum = 0, many = 0;
                for (int r = 0; r < C; ++r) {
                    sum += of(r).hist[tid];
                    many += of(r).count[tid];
                }
                s.list[tid] = sum;
                s.list[tid + 256] = many;
            }
            __syncthreads();
            int d = 255;
            for (; d > 0; --d) {
                if (s.list[256 + d] && (double)(before + s.list[d]) >= limit) break;
                before += s.list[d];
            }
            prefix |= (uint32_t)d << bits;
            here = s.list[256 + d];
            sync();                                    // the sums have been read
        }
        // `here` tokens have this key: as many of them as it takes, the lower indices first
        const float found = logit_of(prefix);
        const uint64_t w = by_weight ? weight(found) : 1;
        const double ties = w ? ceil((limit - (double)before) / (double)w) : (double)here;
        const uint64_t take = ties < 1.0 ? 1 : ties > (double)here ? here : (uint64_t)ties;
        const int n = 4 * fours, each_warp = (n + kSampleThreads - 1) / kSampleThreads * 32, i0 = warp * each_warp, i1 = min(i0 + each_warp, n);
        auto same = [&](int i) { return i < i1 && logits[i] == found && kept(found, base + i); };
        uint64_t mine = 0;
        for (int i = i0; i < i1; i += 32) mine += __popc(__ballot_sync(0xffffffffu, same(i + lane)));
        if (lane == 0) s.red2[warp] = mine;
        __syncthreads();
        uint64_t all = 0, front = 0;
        for (int i = 0; i < kSampleWarps; ++i) {
            if (i == warp) front = all;
            all += s.red2[i];
        }
        if (tid < C) of(tid).share2[me] = all;
        sync();
        for (int r = 0; r < me; ++r) front += s.share2[r];
        if (front < take && take <= front + mine)
            for (int i = i0; i < i1; i += 32) {
                const unsigned b = __ballot_sync(0xffffffffu, same(i + lane));
                if (same(i + lane) && front + __popc(b & ((2u << lane) - 1)) == take)
                    for (int r = 0; r < C; ++r) of(r).border = rank_of(found, base + i + lane);
                front += __popc(b);
            }
    }
};

template <typename T, int C>
__global__ void __launch_bounds__(kSampleThreads, 2) __cluster_dims__(C, 1, 1)
sample_kernel(const __grid_constant__ zkfp_sample_args a, int slice, int vectors)
{
    extern __shared__ __align__(16) float logits[];
    __shared__ SampleShared s;
    chain_enter();
    // nobody touches another CTA's shared memory before that has started
    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const long long row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = C == 1 ? 0 : (int)(blockIdx.x % C), V = (int)a.vocab;
    const int base = me * slice, n = max(0, min(slice, V - base));
    const T* l = (const T*)a.logits + row * a.ld + base;
    const float temperature = a.temperature ? a.temperature[row] : a.value_temperature;
    const int top_k = a.top_k ? a.top_k[row] : a.value_top_k;
    const float top_p = a.top_p ? a.top_p[row] : a.value_top_p, min_p = a.min_p ? a.min_p[row] : a.value_min_p, u = a.random[row];
    if (tid < 256) s.table[tid] = exp2((double)tid / 256.0);
    // the largest logit, and the smallest finite one
    float best = -INFINITY, least = INFINITY;
    auto take = [&](float x) {
        x = plain_logit(x);
        best = fmaxf(best, x);
        least = fminf(least, x == -INFINITY ? INFINITY : x);
        return x;
    };
    const int whole = vectors ? n / 8 * 8 : 0, fours = (n + 3) / 4;
    for (int i = tid * 8; i < whole; i += kSampleThreads * 8) {
        float x[8];
        load8(l + i, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = take(x[k]);
        store8(logits + i, x);
    }
    for (int i = whole + tid; i < 4 * fours; i += kSampleThreads) logits[i] = i < n ? take(to_f32(l[i])) : -INFINITY;
    best = warp_max(best);
    least = -warp_max(-least);
    if (lane == 0) s.red[warp] = (uint64_t)__float_as_uint(best) << 32 | __float_as_uint(least);
    __syncthreads();
    for (int i = 0; i < kSampleWarps; ++i) {
        best = fmaxf(best, __uint_as_float((uint32_t)(s.red[i] >> 32)));
        least = fminf(least, __uint_as_float((uint32_t)s.red[i]));
    }
    Sampler<T, C> p{cg::this_cluster(), s, logits, fours, base, me, tid, lane, warp};
    if (C > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (tid < C) {
            p.of(tid).best[me] = best;
            p.of(tid).least[me] = least;
        }
        p.sync();
        for (int r = 0; r < C; ++r) {
            best = fmaxf(best, s.best[r]);
            least = fminf(least, s.least[r]);
        }
    }
    if (best == -INFINITY) {
        if (tid == 0 && me == 0) a.out[row] = -1;
        return;
    }
    const bool greedy = !(temperature > 0.f);
    if (greedy) {
        uint32_t first = 0xffffffffu;
        for (int i = tid; i < n; i += kSampleThreads)
            if (logits[i] == best) first = min(first, (uint32_t)(base + i));
        first = __reduce_min_sync(0xffffffffu, first);
        __syncthreads();
        if (lane == 0) s.red[warp] = first;
        __syncthreads();
        for (int i = 0; i < kSampleWarps; ++i) first = min(first, (uint32_t)s.red[i]);
        if (tid < C) p.of(tid).first[me] = first;
        p.sync();
        for (int r = 0; r < C; ++r) first = min(first, s.first[r]);
        if (tid == 0 && me == 0) a.out[row] = first;
        return;
    }
    // An infinite largest logit: its like alone are kept, and count as the largest finite number.  exp(-40) is 2^-57.
    const float top = fminf(best, 3.402823466e38f);
    p.weight = Weigher{s.table, (double)top, 256 * 1.4426950408889634 / (double)temperature, top - 40.f * temperature, top};
    p.top = top;
    p.low = best == INFINITY ? top : -INFINITY;                        // no -infinity is kept, whatever becomes of its weight
    p.upto = 0;
    {
        // logits below 2^-46 of the largest weight share the last stretch
        const float span = top - fmaxf(least, top - fminf(32.f * temperature, 3e38f));
        p.per = span > 0.f && span < INFINITY ? (float)kStretches / span : 0.f;
        if (!(p.per < 3e38f)) p.per = 0.f;
    }
    if (top_k > 0 && top_k < V) p.narrow(false, (uint64_t)top_k, 0.0);
    if (top_p < 1.f) p.narrow(true, 0, top_p > 0.f ? (double)top_p : 0.0);
    const double enough = min_p > 0.f ? 256 * fmin(log2((double)min_p), 0.0) : -INFINITY;
    // kept weight by warps, each a stretch of the indices; then the token inside its stretch
    const int each_warp = (fours + kSampleThreads - 1) / kSampleThreads * 32, i0 = warp * each_warp, i1 = min(i0 + each_warp, fours);
    auto four = [&](int i, uint64_t (&w)[4]) {
        const float4 v = *reinterpret_cast<const float4*>(logits + 4 * i);
        const float x[4] = {v.x, v.y, v.z, v.w};
        w[0] = w[1] = w[2] = w[3] = 0;
        // most groups of four of a row that has been narrowed hold nothing
        if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) < p.low) return;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint64_t here = p.weight(x[k]);
            w[k] = p.kept(x[k], base + 4 * i + k) && p.weight.exponent(x[k]) >= enough ? here : 0;
        }
    };
    uint64_t mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) {
        uint64_t w[4];
        four(i, w);
        mine += (w[0] + w[1]) + (w[2] + w[3]);
    }
    mine = warp_add64(mine);
    __syncthreads();
    if (lane == 0) s.red[warp] = mine;
    __syncthreads();
    uint64_t all = 0, front = 0, total = 0;
    for (int i = 0; i < kSampleWarps; ++i) {
        if (i == warp) front = all;
        all += s.red[i];
    }
    if (C > 1) {
        if (tid < C) p.of(tid).share2[me] = all;
        p.sync();
        for (int r = 0; r < C; ++r) {
            if (r < me) front += s.share2[r];
            total += s.share2[r];
        }
    } else {
        total = all;
    }
    // random < 1, so some token passes it; rounding must not take it to the total itself
    const uint64_t target = min((uint64_t)((double)u * (double)total), total - 1);
    if (target < front || target >= front + mine) return;
    for (int i = i0; i < i1; i += 32) {
        uint64_t w[4] = {};
        if (i + lane < i1) four(i + lane, w);
        const uint64_t sum = (w[0] + w[1]) + (w[2] + w[3]), run = warp_scan64(sum);
        const unsigned past = __ballot_sync(0xffffffffu, front + run > target);
        if (past) {
            if (lane == __ffs(past) - 1) {
                uint64_t before = front + run - sum;
                int k = 0;
                while (k < 3 && before + w[k] <= target) before += w[k++];
                a.out[row] = base + 4 * (i + lane) + k;
            }
            return;
        }
        front += __shfl_sync(0xffffffffu, run, 31);
    }
}

template <typename T, int C>
int launch_sample(const zkfp_sample_args& a, cudaStream_t st)
{
    const int slice = (int)((a.vocab + C * 8 - 1) / (C * 8) * 8);
    const int vectors = !((uintptr_t)a.logits & 15) && !(a.ld * (long long)sizeof(T) & 15);
    ZKDS_CUDA(cudaFuncSetAttribute(sample_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax - (int)sizeof(SampleShared) - 1024));
    fp_launch(sample_kernel<T, C>, dim3((unsigned)(a.rows * C)), dim3(kSampleThreads), (size_t)slice * 4, st, a, slice, vectors);
    return fp_launched();
}

template <typename T>
int launch_sample(const zkfp_sample_args& a, cudaStream_t st)
{
    // slices of up to 18000 logits leave room for two CTAs per SM; few rows are cut further, down to 2048
    int c = 1;
    while (c < kClusterMost && (a.vocab > 18000 * c || (a.rows * c < fp_sm_count() && a.vocab > 2048 * c))) c *= 2;
    switch (c) {
    case 1: return launch_sample<T, 1>(a, st);
    case 2: return launch_sample<T, 2>(a, st);
    case 4: return launch_sample<T, 4>(a, st);
    default: return launch_sample<T, 8>(a, st);
    }
}

}  // namespace

}  // namespace zkds

using namespace zkds;

extern "C" int zkfp_sample(const zkfp_sample_args* a, void* stream)
{
    if (!a || !a->logits || !a->random || !a->out || a->rows < 0 || a->vocab <= 0 || a->ld < a->vocab || (unsigned)a->dtype > 1) return ZKDS_ERR_ARG;
    if (a->rows > 0x7fffffffll / kClusterMost || a->vocab > (1 << 18)) return ZKDS_ERR_UNSUPPORTED;
    if (a->rows == 0) return ZKDS_OK;
    return a->dtype == ZKFP_BF16 ? launch_sample<bf16>(*a, (cudaStream_t)stream) : launch_sample<float>(*a, (cudaStream_t)stream);
}
