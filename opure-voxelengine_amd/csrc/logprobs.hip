// ============================================================================
//  logprobs.hip -- log probabilities of given tokens, the entropy and the most
//  probable tokens of rows of logits.
//
//  With y = x / temperature, m = max y, S = sum e^(y - m), E = sum e^(y - m) (y - m):
//    log p(t) = (y_t - m) - log S,   entropy = log S - E / S
//  (both terms of the entropy are positive: nothing cancels).  One pass: a lane
//  holds m, S and E of what it has read; past a new maximum m',
//    S' = S f,  E' = (E + S (m - m')) f,  f = e^(m - m').
//  The largest logits go by a 64-bit key, the value's bits in order above the
//  index's complement, so no two are equal and ties fall to the lowest index.
// ============================================================================
#include "internal.h"

#include <algorithm>

using namespace opure_dev_math;

namespace {

constexpr uint32_t PER = 16;                         // logits a lane holds at a time
constexpr uint32_t CHUNK = 64 * PER;                 // a wave's
constexpr uint32_t MAX_SLICES = 64;
constexpr float NEG_INF = -__builtin_huge_valf();

struct LogprobParams {
    const float* logits;
    const int32_t* tokens;
    float* logprob;
    float* entropy;
    int32_t* top_tokens;
    float* top_logprobs;
    float4* stats;             // [rows][slices]: m, S, E, whether a logit is NaN or +inf
    uint64_t* keys;            // [rows][slices][top]
    uint64_t stride;
    uint32_t rows, vocab, top, slices, slice;        // logits a slice: a multiple of 4 CHUNK
    float temperature;
    uint32_t* err;
};

__device__ __forceinline__ uint32_t order_key(float f)
{
    if (f != f) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(f == 0.0f ? 0.0f : f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k)
{
    return k == 0xFFFFFFFFu ? __builtin_nanf("") : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ uint64_t make_key(float f, uint32_t at) { return static_cast<uint64_t>(order_key(f)) << 32 | (0xFFFFFFFFu - at); }

__device__ __forceinline__ uint64_t lane_xor(uint64_t v, uint32_t x)
{
    return static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(v), static_cast<int>(x)));
}
__device__ __forceinline__ uint64_t pick(uint64_t v, uint64_t o, bool larger) { return (v > o) == larger ? v : o; }

// 64 keys, one a lane, into falling order
__device__ inline uint64_t wave_sort(uint64_t v)
{
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t k = 2; k <= 64u; k <<= 1)
#pragma unroll
        for (uint32_t j = k >> 1; j > 0u; j >>= 1)
            v = pick(v, lane_xor(v, j), ((lane & j) == 0u) == ((lane & k) == 0u || k == 64u));
    return v;
}
// the 64 largest of two falling sequences, falling
__device__ inline uint64_t wave_merge(uint64_t a, uint64_t b)
{
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t r = lane_xor(b, 63u);
    uint64_t v = a > r ? a : r;
#pragma unroll
    for (uint32_t j = 32; j > 0u; j >>= 1) v = pick(v, lane_xor(v, j), (lane & j) == 0u);
    return v;
}
__device__ __forceinline__ uint64_t key_at(uint64_t v, uint32_t lane)
{
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(lane)));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), static_cast<int>(lane)));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

struct Stats {
    float m, s, e;
    bool bad;
};

// f (S and E) to a maximum m2 >= m
__device__ __forceinline__ void rebase(Stats& a, float m2)
{
    const bool none = a.m == NEG_INF;
    const float d = none ? 0.0f : __fsub_rn(a.m, m2), f = __builtin_amdgcn_exp2f(__fmul_rn(d, 1.44269504088896340736f));
    a.e = __fmul_rn(__fmaf_rn(a.s, d, a.e), f);
    a.s = __fmul_rn(a.s, f);
    a.m = m2;
}

__device__ __forceinline__ Stats wave_stats(Stats a)
{
    rebase(a, wave_max64(a.m));
    a.s = wave_sum64(a.s);
    a.e = wave_sum64(a.e);
    a.bad = __any(a.bad);
    return a;
}

// A row's results from its sums and its largest keys, by one wave.
__device__ __forceinline__ void finish(const LogprobParams& p, uint32_t row, Stats a, uint64_t best)
{
    const uint32_t lane = threadIdx.x & 63u;
    const float nan = __builtin_nanf("");
    const bool bad = a.bad || a.s == 0.0f;
    const float norm = logf(a.s);
    auto of = [&](float x) { return bad ? nan : __fsub_rn(__fsub_rn(p.temperature == 1.0f ? x : __fdiv_rn(x, p.temperature), a.m), norm); };
    if (lane == 0u && p.entropy) p.entropy[row] = bad ? nan : __fsub_rn(norm, __fdiv_rn(a.e, a.s));
    if (lane == 0u && p.logprob)
    {
        const int32_t t = p.tokens[row];
        const bool in = t >= 0 && static_cast<uint32_t>(t) < p.vocab;
        if (!in) p.err[ERR_TOKEN] = 1u;
        p.logprob[row] = in ? of(p.logits[row * p.stride + static_cast<uint32_t>(t)]) : nan;
    }
    if (lane < p.top)
    {
        const uint64_t at = static_cast<uint64_t>(row) * p.top + lane;
        p.top_tokens[at] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
        p.top_logprobs[at] = of(key_value(static_cast<uint32_t>(best >> 32)));
    }
}

// A slice of a row by a workgroup, its waves every fourth chunk.  A wave keeps its
// 64 largest keys in order, one a lane; of a logit only a comparison with the
// top-th of them is needed, and the few that pass wait in LDS until they are 64.
// The first chunk's lanes' maxima are the first 64.
template <bool TOP, bool ONE>
__global__ __launch_bounds__(256) void k_logprobs(LogprobParams p)
{
    __shared__ uint64_t queue[TOP ? 4 : 1][TOP ? 128 : 1];
    __shared__ float4 part[4];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t row = blockIdx.x / p.slices, sl = blockIdx.x - row * p.slices;
    const float* x = p.logits + row * p.stride;
    const uint32_t begin = sl * p.slice, end = min(begin + p.slice, p.vocab);
    const float tau = p.temperature;
    Stats a{NEG_INF, 0.0f, 0.0f, false};
    uint64_t best = 0, least = 0;                        // the lane's key; the top-th
    float bar = NEG_INF;                                 // its value
    uint32_t waiting = 0;
    auto take = [&](uint64_t batch) {
        best = wave_merge(best, wave_sort(batch));
        least = key_at(best, p.top - 1u);
        bar = least ? key_value(static_cast<uint32_t>(least >> 32)) : NEG_INF;
    };
    for (uint32_t c0 = begin + wave * CHUNK; c0 < end; c0 += 4u * CHUNK)
    {
        float v[PER];
        const bool whole = c0 + CHUNK <= end;
#pragma unroll
        for (uint32_t i = 0; i < PER; i += 4u)
        {
            const uint32_t at = c0 + 64u * i + 4u * lane;
            if (whole) __builtin_memcpy(&v[i], x + at, 16);
            else
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) v[i + e] = at + e < end ? x[at + e] : NEG_INF;
        }
        auto index = [&](uint32_t i) { return c0 + 64u * (i & ~3u) + 4u * lane + (i & 3u); };
        if constexpr (TOP)
        {
            uint64_t mine = 0;                           // the lane's largest of the first chunk
            if (c0 < begin + 4u * CHUNK)
            {
#pragma unroll
                for (uint32_t i = 0; i < PER; ++i)
                {
                    const uint64_t k = index(i) < end ? make_key(v[i], index(i)) : 0u;
                    mine = mine > k ? mine : k;
                }
                take(mine);
            }
#pragma unroll
            for (uint32_t i = 0; i < PER; ++i)
            {
                if (!__any(!(v[i] < bar))) continue;
                uint64_t k = index(i) < end ? make_key(v[i], index(i)) : 0u;
                if (k == mine) k = 0u;
                const uint64_t pass = __ballot(k > least);
                if (!pass) continue;
                if (k > least) queue[wave][waiting + __popcll(pass & ((1ull << lane) - 1u))] = k;
                waiting += static_cast<uint32_t>(__popcll(pass));
                if (waiting >= 64u)
                {
                    __builtin_amdgcn_wave_barrier();
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    const uint64_t batch = queue[wave][lane], rest = queue[wave][64u + lane];
                    take(batch);
                    waiting -= 64u;
                    __builtin_amdgcn_wave_barrier();
                    if (lane < waiting) queue[wave][lane] = rest;
                }
            }
        }
        float m = NEG_INF;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i)
        {
            if (tau != 1.0f) v[i] = __fdiv_rn(v[i], tau);
            a.bad = a.bad || !(v[i] < __builtin_huge_valf());
            m = fmaxf(m, v[i]);
        }
        if (m > a.m) rebase(a, m);
        const float ms = a.m == NEG_INF ? 0.0f : a.m;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i)
        {
            // of a masked logit e is 0 and d finite
            const float d = fmaxf(__fsub_rn(v[i], ms), -1e30f), e = __builtin_amdgcn_exp2f(__fmul_rn(d, 1.44269504088896340736f));
            a.s += e;
            a.e = __fmaf_rn(e, d, a.e);
        }
    }
    a = wave_stats(a);
    if constexpr (TOP)
    {
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (waiting) take(lane < waiting ? queue[wave][lane] : 0u);
        __builtin_amdgcn_wave_barrier();
        queue[wave][lane] = best;
    }
    if (lane == 0u) part[wave] = float4{a.m, a.s, a.e, a.bad ? 1.0f : 0.0f};
    __syncthreads();
    if (wave != 0u) return;
    const float4 mine = part[lane & 3u];
    a = wave_stats(Stats{lane < 4u ? mine.x : NEG_INF, lane < 4u ? mine.y : 0.0f, lane < 4u ? mine.z : 0.0f, lane < 4u && mine.w != 0.0f});
    if constexpr (TOP)
#pragma unroll
        for (uint32_t w = 1; w < 4; ++w) best = wave_merge(best, queue[w][lane]);
    if constexpr (ONE) finish(p, row, a, best);
    else
    {
        if (lane == 0u) p.stats[blockIdx.x] = float4{a.m, a.s, a.e, a.bad ? 1.0f : 0.0f};
        if (TOP && lane < p.top) p.keys[static_cast<uint64_t>(blockIdx.x) * p.top + lane] = best;
    }
}

// Joins a row's slices: each of four waves every fourth slice's keys, then the waves'.
template <bool TOP>
__global__ __launch_bounds__(256) void k_logprobs_join(LogprobParams p)
{
    __shared__ uint64_t list[4][64];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, row = blockIdx.x;
    const uint64_t at = static_cast<uint64_t>(row) * p.slices;
    uint64_t best = 0;
    if constexpr (TOP)
    {
        for (uint32_t s = wave; s < p.slices; s += 4u)
        {
            const uint64_t k = lane < p.top ? p.keys[(at + s) * p.top + lane] : 0u;
            best = s == wave ? k : wave_merge(best, k);
        }
        list[wave][lane] = best;
        __syncthreads();
    }
    if (wave != 0u) return;
    if constexpr (TOP)
#pragma unroll
        for (uint32_t w = 1; w < 4; ++w) best = wave_merge(best, list[w][lane]);
    const float4 mine = p.stats[at + min(lane, p.slices - 1u)];
    const bool in = lane < p.slices;
    finish(p, row, wave_stats(Stats{in ? mine.x : NEG_INF, in ? mine.y : 0.0f, in ? mine.z : 0.0f, in && mine.w != 0.0f}), best);
}

// A row in as many slices as give each CU two workgroups.
void slices_of(const opure_dev* dev, const opure_logprobs_args* a, uint32_t& slices, uint32_t& slice)
{
    const uint32_t cu = dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u, most = (a->vocab + 4u * CHUNK - 1u) / (4u * CHUNK);
    slices = std::min({std::max(1u, 2u * cu / a->rows), most, MAX_SLICES});
    slice = ((a->vocab + slices - 1u) / slices + 4u * CHUNK - 1u) / (4u * CHUNK) * (4u * CHUNK);
    slices = (a->vocab + slice - 1u) / slice;
}

uint64_t stats_bytes(const opure_logprobs_args* a, uint32_t slices)
{
    return slices > 1u ? opure_hip::align_up(static_cast<uint64_t>(a->rows) * slices * 16u, 256) : 0u;
}
uint64_t key_bytes(const opure_logprobs_args* a, uint32_t slices)
{
    return slices > 1u ? static_cast<uint64_t>(a->rows) * slices * a->top * 8u : 0u;
}

int shape_validate(const opure_logprobs_args* a)
{
    OPURE_REQUIRE(a, OPURE_E_INVALID, "opure_logprobs: null argument");
    OPURE_REQUIRE(a->rows >= 1 && a->rows <= OPURE_MAX_LOGPROB_ROWS, OPURE_E_CAPACITY, "opure_logprobs: %u rows outside 1..%d", a->rows,
                  OPURE_MAX_LOGPROB_ROWS);
    OPURE_REQUIRE(a->vocab >= 1 && a->vocab <= 1u << 24, OPURE_E_CAPACITY, "opure_logprobs: vocab %u outside 1..2^24", a->vocab);
    OPURE_REQUIRE(a->top <= OPURE_MAX_TOP && a->top <= a->vocab, OPURE_E_CAPACITY, "opure_logprobs: top %u beyond %d or vocab %u", a->top,
                  OPURE_MAX_TOP, a->vocab);
    return OPURE_OK;
}

}  // namespace

using namespace opure_hip;

extern "C" int opure_logprobs_reserve(opure_dev* dev, const opure_logprobs_args* a)
{
    OPURE_REQUIRE(dev, OPURE_E_INVALID, "opure_logprobs_reserve: null device");
    const int rc = shape_validate(a);
    if (rc) return rc;
    const DeviceGuard on(dev);
    uint32_t slices, slice;
    slices_of(dev, a, slices, slice);
    return ensure_workspace(dev, stats_bytes(a, slices) + key_bytes(a, slices));
}

extern "C" int opure_logprobs(opure_dev* dev, const opure_logprobs_args* a)
{
    OPURE_REQUIRE(dev && a && a->logits, OPURE_E_INVALID, "opure_logprobs: null argument");
    const int rv = shape_validate(a);
    if (rv) return rv;
    OPURE_REQUIRE((a->tokens != nullptr) == (a->logprob != nullptr), OPURE_E_INVALID, "opure_logprobs: tokens and logprob come together");
    OPURE_REQUIRE((a->top != 0u) == (a->top_tokens != nullptr) && (a->top != 0u) == (a->top_logprobs != nullptr), OPURE_E_INVALID,
                  "opure_logprobs: top %u, top_tokens and top_logprobs come together", a->top);
    OPURE_REQUIRE(a->logprob || a->entropy || a->top, OPURE_E_INVALID, "opure_logprobs: nothing asked for");
    OPURE_REQUIRE(a->temperature > 0.0f && a->temperature < __builtin_huge_valf(), OPURE_E_INVALID, "opure_logprobs: temperature must be positive");
    OPURE_REQUIRE(a->logits_stride >= a->vocab, OPURE_E_INVALID, "opure_logprobs: logits_stride %u below vocab %u", a->logits_stride, a->vocab);
    auto address = [](const void* at) { return reinterpret_cast<uintptr_t>(at); };
    OPURE_REQUIRE(((address(a->logits) | address(a->tokens) | address(a->logprob) | address(a->entropy) | address(a->top_tokens) |
                    address(a->top_logprobs)) & 3u) == 0u, OPURE_E_INVALID, "opure_logprobs: pointers must be 4-byte aligned");
    const uint64_t logits = (static_cast<uint64_t>(a->rows - 1u) * a->logits_stride + a->vocab) * 4u, one = a->rows * 4ull, tops = one * a->top;
    const struct { const char* name; const void* at; uint64_t bytes; } part[] = {
        {"logprob", a->logprob, one}, {"entropy", a->entropy, one}, {"top_tokens", a->top_tokens, tops}, {"top_logprobs", a->top_logprobs, tops},
        {"logits", a->logits, logits}, {"tokens", a->tokens, one}, {"the device's workspace", dev->ws, dev->ws_bytes}};
    for (int x = 0; x < 4; ++x)
        for (int y = x + 1; y < 7; ++y)
            OPURE_REQUIRE(!overlaps(part[x].at, part[x].bytes, part[y].at, part[y].bytes), OPURE_E_INVALID, "opure_logprobs: %s overlaps %s",
                          part[x].name, part[y].name);
    const DeviceGuard on(dev);
    LogprobParams p{};
    slices_of(dev, a, p.slices, p.slice);
    const uint64_t stats = stats_bytes(a, p.slices), bytes = stats + key_bytes(a, p.slices);
    // the workspace may move, and the slices' results go there
    OPURE_REQUIRE(!bytes || (!overlaps(dev->ws, dev->ws_bytes, a->logits, logits) && !overlaps(dev->ws, dev->ws_bytes, a->tokens, one)),
                  OPURE_E_INVALID, "opure_logprobs: logits or tokens in the device's workspace");
    if (bytes)
    {
        const int rc = ensure_workspace(dev, bytes);
        if (rc) return rc;
    }
    p.logits = a->logits;
    p.tokens = a->tokens;
    p.logprob = a->logprob;
    p.entropy = a->entropy;
    p.top_tokens = a->top_tokens;
    p.top_logprobs = a->top_logprobs;
    p.stats = static_cast<float4*>(dev->ws);
    p.keys = bytes ? reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(dev->ws) + stats) : nullptr;
    p.stride = a->logits_stride;
    p.rows = a->rows;
    p.vocab = a->vocab;
    p.top = a->top;
    p.temperature = a->temperature;
    p.err = dev->err;
    const dim3 grid(p.rows * p.slices), block(256);
    if (p.slices == 1u)
    {
        if (p.top) OPURE_LAUNCH(dev, (k_logprobs<true, true>), grid, block, 0, p);
        else OPURE_LAUNCH(dev, (k_logprobs<false, true>), grid, block, 0, p);
        OPURE_LAUNCH_CHECK("k_logprobs");
        return OPURE_OK;
    }
    if (p.top) OPURE_LAUNCH(dev, (k_logprobs<true, false>), grid, block, 0, p);
    else OPURE_LAUNCH(dev, (k_logprobs<false, false>), grid, block, 0, p);
    OPURE_LAUNCH_CHECK("k_logprobs");
    if (p.top) OPURE_LAUNCH(dev, (k_logprobs_join<true>), dim3(p.rows), block, 0, p);
    else OPURE_LAUNCH(dev, (k_logprobs_join<false>), dim3(p.rows), block, 0, p);
    OPURE_LAUNCH_CHECK("k_logprobs_join");
    return OPURE_OK;
}
