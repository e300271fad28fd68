// One token per row of logits from given random numbers: temperature, the k largest, the likeliest p, at least min_p.
//
// Weights are w = 2^((l - max) log2(e) / temperature), held as whole multiples of 2^-44: their sums are exact in any order,
// so that neither the threads' timing nor the shape of the launch moves a border between two tokens.  2^y is made in 64
// bits: y by one product, 2^y from a table of 2^(i / 256) and the series of 2^r, |r| <= 1 / 512, to its fifth term (the sixth
// is 2^-57 of it).
//
// What a row keeps is a prefix of its tokens in falling order of (logit, then rising index): the threshold is found on the logits'
// bits, ordered as whole numbers, 8 of 32 bits at a time: how many tokens, or how much weight, lies in each of the 256
// continuations of the bits found so far.
#include "float_common.cuh"

namespace zkds {

namespace {

constexpr int kSampleThreads = 512;
constexpr double kWeightOne = 17592186044416.0;        // 2^44

// larger logits have larger keys; NaN the key of -infinity
__device__ __forceinline__ uint32_t key_of(float l)
{
    if (l != l) l = -INFINITY;
    if (l == 0.f) l = 0.f;                             // both zeros are equal
    const uint32_t u = __float_as_uint(l);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Weigher {
    const double* table;             // 2^(i / 256) 2^44
    double top, scale;
    bool infinite;                   // the largest logit is: its like have weight 1, all others none
    __device__ __forceinline__ double exponent(float l) const
    {
        return infinite ? (l == INFINITY ? 0.0 : -100.0) : ((double)l - top) * scale;
    }
    __device__ __forceinline__ uint64_t operator()(uint32_t key) const
    {
        const double y = exponent(logit_of(key));
        if (!(y > -46.0)) return 0;
        const double n = rint(y * 256.0);
        const double r = (y - n * 0.00390625) * 0.6931471805599453;
        const int i = (int)n;
        const double e = 1.0 + r * (1.0 + r * (0.5 + r * (1.0 / 6 + r * (1.0 / 24 + r * (1.0 / 120)))));
        return (uint64_t)(ldexp(table[i & 255] * e, i >> 8) + 0.5);
    }
};

__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t* red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < kSampleThreads / 32; ++i) t += red[i];
    return t;
}

// The smallest prefix in falling order that is complete: `wanted` tokens, or tokens until the weight in front reaches `mass`.  In:
// what a row keeps so far (keys above `low`, and the first `ties` equal to it).  Out: the same of the prefix.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads)
sample_kernel(const zkfp_sample_args a)
{
    chain_enter();
    __shared__ double table[256];
    __shared__ unsigned long long mass[256];
    __shared__ unsigned count[256];
    __shared__ uint64_t red[kSampleThreads / 32], red2[kSampleThreads / 32];
    __shared__ unsigned s_key;
    __shared__ unsigned long long s_mass, s_count;
    const long long row = blockIdx.x;
    const T* l = (const T*)a.logits + row * a.ld;
    const int V = (int)a.vocab, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float temperature = a.temperature ? a.temperature[row] : a.value_temperature;
    const int top_k = a.top_k ? a.top_k[row] : a.value_top_k;
    const float top_p = a.top_p ? a.top_p[row] : a.value_top_p, min_p = a.min_p ? a.min_p[row] : a.value_min_p;
    if (tid < 256) table[tid] = exp2((double)tid / 256.0) * kWeightOne;
    uint32_t best = 0;
    for (int i = tid; i < V; i += kSampleThreads) best = max(best, key_of(to_f32(l[i])));
    best = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) red[warp] = best;
    __syncthreads();
    for (int i = 0; i < kSampleThreads / 32; ++i) best = max(best, (uint32_t)red[i]);
    const float top = logit_of(best);
    if (top == -INFINITY) {
        if (tid == 0) a.out[row] = -1;
        return;
    }
    const bool greedy = !(temperature > 0.f);
    const Weigher weight{table, (double)top, greedy ? 0.0 : 1.4426950408889634 / (double)temperature, top == INFINITY};
    uint32_t low = 0;
    unsigned long long ties = V;               // kept: keys above low, and the first `ties` equal to it
    // finds the prefix; by count if by_mass is false
    auto narrow = [&](bool by_mass, unsigned long long wanted, double limit) {
        const uint32_t floor_key = low;
        const unsigned long long floor_ties = ties;
        uint32_t prefix = 0;
        unsigned long long before_mass = 0, before_count = 0;        // of keys above the bits found so far
        for (int bits = 24; bits >= 0; bits -= 8) {
            __syncthreads();
            if (tid < 256) { mass[tid] = 0; count[tid] = 0; }
            __syncthreads();
            for (int i = tid; i < V; i += kSampleThreads) {
                const uint32_t k = key_of(to_f32(l[i]));
                if (k < floor_key || (bits < 24 && (k >> (bits + 8)) != (prefix >> (bits + 8)))) continue;
                atomicAdd(&count[(k >> bits) & 255], 1u);
                if (by_mass) atomicAdd(&mass[(k >> bits) & 255], (unsigned long long)weight(k));
            }
            __syncthreads();
            if (tid == 0) {
                int bin = 255;
                for (; bin > 0; --bin) {
                    const bool done = by_mass ? (double)(before_mass + mass[bin]) >= limit : before_count + count[bin] >= wanted;
                    if (count[bin] && done) break;
                    before_mass += mass[bin];
                    before_count += count[bin];
                }
                s_key = prefix | ((uint32_t)bin << bits);
                s_mass = before_mass;
                s_count = before_count;
            }
            __syncthreads();
            prefix = s_key;
            before_mass = s_mass;
            before_count = s_count;
        }
        // all keys equal to prefix: how many of them
        const unsigned long long here = count[prefix & 255];
        unsigned long long n;
        if (by_mass) {
            const double w = (double)weight(prefix), rest = limit - (double)before_mass;
            n = w > 0.0 ? (unsigned long long)fmin(ceil(rest / w), (double)here) : here;
            if (n < 1) n = 1;
        } else {
            n = min(wanted - before_count, here);
        }
        if (prefix == floor_key) n = min(n, floor_ties);
        low = prefix;
        ties = n;
    };
    if (greedy) {
        low = best;
        ties = 1;
    } else {
        if (top_k > 0 && top_k < V) narrow(false, (unsigned long long)top_k, 0.0);
        if (top_p < 1.f) {
            uint64_t m = 0, t = 0;
            for (int i = tid; i < V; i += kSampleThreads) {
                const uint32_t k = key_of(to_f32(l[i]));
                if (k > low) m += weight(k);
                else if (k == low) ++t;
            }
            m = block_sum64(m, red);
            t = block_sum64(t, red2);
            m += min((unsigned long long)t, ties) * weight(low);
            narrow(true, 0, (double)(top_p > 0.f ? top_p : 0.f) * (double)m);
        }
        if (min_p > 0.f) {
            // the smallest key that is likely enough
            const double least = fmin(log2((double)min_p), 0.0);
            uint32_t lowest = 0xffffffffu;
            for (int i = tid; i < V; i += kSampleThreads) {
                const uint32_t k = key_of(to_f32(l[i]));
                if (weight.exponent(logit_of(k)) >= least) lowest = min(lowest, k);
            }
            lowest = __reduce_min_sync(0xffffffffu, lowest);
            __syncthreads();
            if (lane == 0) red[warp] = lowest;
            __syncthreads();
            for (int i = 0; i < kSampleThreads / 32; ++i) lowest = min(lowest, (uint32_t)red[i]);
            if (lowest > low) {
                low = lowest;
                ties = V;
            }
        }
    }
    // kept weight by warps, each a stretch of the indices; then the token inside its stretch
    const int stretch = (V + kSampleThreads - 1) / kSampleThreads * 32, i0 = warp * stretch, i1 = min(i0 + stretch, V);
    uint64_t above = 0, equal = 0;
    for (int i = i0 + lane; i < i1; i += 32) {
        const uint32_t k = key_of(to_f32(l[i]));
        if (k > low) above += weight(k);
        else if (k == low) ++equal;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        above += __shfl_xor_sync(0xffffffffu, above, o);
        equal += __shfl_xor_sync(0xffffffffu, equal, o);
    }
    __syncthreads();
    if (lane == 0) { red[warp] = above; red2[warp] = equal; }
    __syncthreads();
    const uint64_t w_low = weight(low);
    uint64_t total = 0, mine = 0, mine_ties = 0, seen = 0;           // in front of this warp's stretch
    for (int i = 0; i < kSampleThreads / 32; ++i) {
        if (i == warp) { mine = total; mine_ties = seen; }
        const uint64_t here = seen >= ties ? 0 : min((uint64_t)(ties - seen), red2[i]);
        total += red[i] + here * w_low;
        seen += red2[i];
    }
    // random < 1, so some token passes it; rounding must not take it to the total itself
    const uint64_t target = min((uint64_t)((double)a.random[row] * (double)total), total - 1);
    const uint64_t kept = mine_ties >= ties ? 0 : min((uint64_t)(ties - mine_ties), equal);
    if (target < mine || target >= mine + above + kept * w_low) return;
    uint64_t sum = mine, tie = mine_ties;
    for (int i = i0; i < i1; i += 32) {
        const uint32_t k = i + lane < i1 ? key_of(to_f32(l[i + lane])) : 0;
        const unsigned same = __ballot_sync(0xffffffffu, i + lane < i1 && k == low);
        const bool keep = i + lane < i1 && (k > low || (k == low && tie + __popc(same & ((1u << lane) - 1)) < ties));
        uint64_t v = keep ? weight(k) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum + v > target);
        if (past) {
            if (lane == 0) a.out[row] = i + __ffs(past) - 1;
            return;
        }
        sum += __shfl_sync(0xffffffffu, v, 31);
        tie += __popc(same);
    }
}

}  // namespace

}  // namespace zkds

using namespace zkds;

extern "C" int zkfp_sample(const zkfp_sample_args* a, void* stream)
{
    if (!a || !a->logits || !a->random || !a->out || a->rows < 0 || a->vocab <= 0 || a->ld < a->vocab || (unsigned)a->dtype > 1) return ZKDS_ERR_ARG;
    if (a->rows > 0x7fffffffll || a->vocab > (1 << 18)) return ZKDS_ERR_UNSUPPORTED;
    if (a->rows == 0) return ZKDS_OK;
    if (a->dtype == ZKFP_BF16) fp_launch(sample_kernel<bf16>, dim3((unsigned)a->rows), dim3(kSampleThreads), 0, (cudaStream_t)stream, *a);
    else fp_launch(sample_kernel<float>, dim3((unsigned)a->rows), dim3(kSampleThreads), 0, (cudaStream_t)stream, *a);
    return fp_launched();
}
