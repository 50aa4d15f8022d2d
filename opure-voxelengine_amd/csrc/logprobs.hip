// ============================================================================
//  logprobs.hip -- log probabilities of given tokens, the entropy and the most
//  probable tokens of rows of logits.
//
//  With m = max x, d = (x - m) / temperature, S = sum e^d, E = sum e^d d:
//    log p(t) = d_t - log S,   entropy = log S - E / S
//  (both terms of the entropy are positive: nothing cancels).  x / temperature itself
//  may pass fp32's numbers below a temperature of 1, of a row's largest or of all of a
//  row that a mask has at the type's lowest value.  One pass: a lane
//  holds m, S and E of what it has read; past a new maximum m', c = (m - m') / temperature,
//    S' = S f,  E' = (E + S c) f,  f = e^c.
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

// Lanes l and l ^ J exchange keys: the larger goes to the lanes of UP.  All moves are
// the vector unit's (DPP, and the swaps of 16 and 32 lanes, which leave both keys in
// both lanes): a step is about 8 instructions, a fifth of one through LDS.
template <uint32_t J, uint64_t UP>
__device__ __forceinline__ uint64_t exchange(uint64_t v)
{
    uint32_t lo = static_cast<uint32_t>(v), hi = static_cast<uint32_t>(v >> 32), lo2, hi2;
    if constexpr (J >= 16u)
    {
        const auto l = J == 32u ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false) : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
        const auto h = J == 32u ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false) : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
        lo = l[0], lo2 = l[1], hi = h[0], hi2 = h[1];
    }
    else
    {
        // quad_perm [1,0,3,2] and [2,3,0,1], row_ror:8; 4: the half rows mirrored, then the quads
        constexpr int CTRL = J == 1u ? 0xB1 : J == 2u ? 0x4E : J == 8u ? 0x128 : 0x141;
        lo2 = __builtin_amdgcn_mov_dpp(static_cast<int>(lo), CTRL, 0xF, 0xF, true);
        hi2 = __builtin_amdgcn_mov_dpp(static_cast<int>(hi), CTRL, 0xF, 0xF, true);
        if constexpr (J == 4u)
        {
            lo2 = __builtin_amdgcn_mov_dpp(static_cast<int>(lo2), 0x1B, 0xF, 0xF, true);
            hi2 = __builtin_amdgcn_mov_dpp(static_cast<int>(hi2), 0x1B, 0xF, 0xF, true);
        }
    }
    const uint64_t a = static_cast<uint64_t>(hi) << 32 | lo, b = static_cast<uint64_t>(hi2) << 32 | lo2;
    return (a > b) == __builtin_amdgcn_inverse_ballot_w64(UP) ? a : b;
}

// lanes whose bit J is 0 where bit K is 0 (K 64: everywhere), and the others
constexpr uint64_t lanes_up(uint32_t j, uint32_t k)
{
    uint64_t m = 0;
    for (uint32_t l = 0; l < 64u; ++l) m |= static_cast<uint64_t>(((l & j) == 0u) == ((l & k) == 0u)) << l;
    return m;
}
template <uint32_t J, uint32_t K, bool FALLING>
__device__ __forceinline__ uint64_t steps(uint64_t v)
{
    v = exchange<J, FALLING ? lanes_up(J, K) : ~lanes_up(J, K)>(v);
    if constexpr (J > 1u) return steps<J / 2u, K, FALLING>(v);
    else return v;
}
// 64 keys, one a lane, into rising order
template <uint32_t K = 2>
__device__ __forceinline__ uint64_t wave_sort(uint64_t v)
{
    v = steps<K / 2u, K, false>(v);
    if constexpr (K < 64u) return wave_sort<2u * K>(v);
    else return v;
}
// the 64 largest of a falling and a rising sequence, falling
__device__ __forceinline__ uint64_t wave_merge(uint64_t falling, uint64_t rising) { return steps<32, 64, true>(falling > rising ? falling : rising); }

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

constexpr float LEAST = -1e30f;                      // of d: e^d is 0 long before, and 2^24 of them have a finite sum

__device__ __forceinline__ float over(float d, float tau) { return __builtin_expect(tau == 1.0f, 1) ? d : __fdiv_rn(d, tau); }

// f (S and E) to a maximum m2 >= m.  Logits that a mask has at the type's lowest value are such a step below.
__device__ __forceinline__ void rebase(Stats& a, float m2, float tau)
{
    const bool none = a.m == NEG_INF;
    const float d = none ? 0.0f : fmaxf(over(__fsub_rn(a.m, m2), tau), LEAST), f = __builtin_amdgcn_exp2f(__fmul_rn(d, 1.44269504088896340736f));
    a.e = __fmul_rn(__fmaf_rn(a.s, d, a.e), f);
    a.s = __fmul_rn(a.s, f);
    a.m = m2;
}

__device__ __forceinline__ Stats wave_stats(Stats a, float tau)
{
    rebase(a, wave_max64(a.m), tau);
    a.s = wave_sum64(a.s);
    a.e = wave_sum64(a.e);
    a.bad = __any(a.bad);
    return a;
}

// A row's token and its logit, asked for before the sums are there.
struct Given {
    bool in;
    float x;
    __device__ __forceinline__ Given(const LogprobParams& p, uint32_t row) : in(false), x(0.0f)
    {
        if (!p.logprob) return;
        const int32_t t = p.tokens[row];
        in = t >= 0 && static_cast<uint32_t>(t) < p.vocab;
        x = p.logits[row * p.stride + (in ? static_cast<uint32_t>(t) : 0u)];
    }
};

// A row's results from its sums and its largest keys, by one wave.
__device__ __forceinline__ void finish(const LogprobParams& p, uint32_t row, Stats a, uint64_t best, const Given& given)
{
    const uint32_t lane = threadIdx.x & 63u;
    const float nan = __builtin_nanf("");
    const bool bad = a.bad || a.s == 0.0f;
    const float norm = logf(a.s);
    // of halves: a temperature brings a difference past fp32's numbers back
    auto of = [&](float x) { return bad ? nan : __fmaf_rn(2.0f, over(__fsub_rn(__fmul_rn(0.5f, x), __fmul_rn(0.5f, a.m)), p.temperature), -norm); };
    if (lane == 0u && p.entropy) p.entropy[row] = bad ? nan : __fsub_rn(norm, __fdiv_rn(a.e, a.s));
    if (lane == 0u && p.logprob)
    {
        if (!given.in) p.err[ERR_TOKEN] = 1u;
        p.logprob[row] = given.in ? of(given.x) : nan;
    }
    if (lane < p.top)
    {
        const uint64_t at = static_cast<uint64_t>(row) * p.top + lane;
        p.top_tokens[at] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
        p.top_logprobs[at] = of(key_value(static_cast<uint32_t>(best >> 32)));
    }
}

// A slice of a row by a workgroup, its waves every fourth chunk.  A wave keeps its 64
// largest keys in order, one a lane.  The first chunk's lanes' maxima are the first 64, so
// at most 16 top logits of it follow; of a later chunk only the lanes' maxima are compared
// with the top-th (an equal logit that comes later loses).  Where one passes, the chunk
// is left in LDS and looked through behind its sums, four logits a lane at a time; those
// that pass go to a queue that is sorted and merged 64 at a time.  Neither the chunk's
// registers nor more than one sort are there for the rare case: with both in the loop the
// compiler took 64 to 135 registers, and 1,500 rows of 128,256 200 us for 158.
//   Bound by memory there: 770 MB in 145 us, 5.3 TB/s.  Few rows are launches, round trips
// and the sorts' chains: one row of 128,256 with its 20 largest 12.3 us, without 7.5.  No
// sorts but each key's place by counting the larger ones took 13.7 and 18.5 (64 largest; 14.3).
template <bool TOP, bool ONE>
__global__ __launch_bounds__(256) void k_logprobs(LogprobParams p)
{
    constexpr uint32_t ROOM = 320;
    __shared__ uint64_t queue[TOP ? 4 : 1][TOP ? ROOM : 1];
    __shared__ float4 chunk[TOP ? 4 : 1][TOP ? PER / 4u : 1u][64];
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
    const uint32_t first = begin + wave * CHUNK;
    for (uint32_t c0 = first; c0 < end; c0 += 4u * CHUNK)
    {
        float v[PER], m = NEG_INF;
        bool bad = false, look = false;
#pragma unroll
        for (uint32_t i = 0; i < PER; i += 4u)
        {
            const uint32_t at = c0 + 64u * i + 4u * lane;
            if (c0 + CHUNK <= end) __builtin_memcpy(&v[i], x + at, 16);
            else
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) v[i + e] = at + e < end ? x[at + e] : NEG_INF;
        }
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i)
        {
            bad = bad || !(v[i] < __builtin_huge_valf());
            m = fmaxf(m, v[i]);
        }
        auto index = [&](uint32_t q) { return c0 + 256u * q + 4u * lane; };
        uint32_t taken = PER;                            // the lane's largest of the first chunk: its first NaN, or m
        float most = m;
        if constexpr (TOP)
        {
            look = c0 == first || __any(bad || m > bar) || (waiting && c0 + 4u * CHUNK >= end);
            if (look)
#pragma unroll
                for (uint32_t q = 0; q < PER / 4u; ++q) chunk[wave][q][lane] = float4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            if (c0 == first)
            {
                bool nan = false;
#pragma unroll
                for (uint32_t i = PER; i-- > 0u;)
                {
                    taken = v[i] == m && !nan ? i : taken;
                    if (v[i] != v[i]) taken = i, nan = true;
                }
                if (nan) most = __builtin_nanf("");
            }
        }
        a.bad = a.bad || bad;
        if (m > a.m) rebase(a, m, tau);
        float ms = a.m == NEG_INF ? 0.0f : a.m;
        if (__builtin_expect(tau != 1.0f, 0))
        {
#pragma unroll
            for (uint32_t i = 0; i < PER; ++i) v[i] = __fdiv_rn(__fsub_rn(v[i], ms), tau);
            ms = 0.0f;
        }
        // a chunk's by themselves: errors of 5.6e-8 on rows of 128,256, of one chain through a lane's 501 logits 2.1e-7
        float cs = 0.0f, ce = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i)
        {
            // of a masked logit e is 0 and d finite
            const float d = fmaxf(__fsub_rn(v[i], ms), LEAST), e = __builtin_amdgcn_exp2f(__fmul_rn(d, 1.44269504088896340736f));
            cs += e;
            ce = __fmaf_rn(e, d, ce);
        }
        a.s += cs;
        a.e += ce;
        if constexpr (TOP)
            if (look)
            {
                // -1: the first chunk's maxima; then four logits of each lane.  Behind them `top` that wait are merged, so that
                // the next chunks are compared with what is largest now, and at the end all
                const uint32_t enough = c0 + 4u * CHUNK >= end ? 1u : min(p.top, 64u);
#pragma unroll 1
                for (int q = c0 == first ? -1 : 0; q < static_cast<int>(PER / 4u); ++q)
                {
                    __builtin_amdgcn_wave_barrier();
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    if (q < 0)
                    {
                        const uint32_t at = index(taken >> 2) + (taken & 3u);
                        queue[wave][lane] = taken < PER && at < end ? make_key(most, at) : 0u;
                        waiting = 64u;
                    }
                    else
                    {
                        const float4 w = chunk[wave][q][lane];
                        const float f[4] = {w.x, w.y, w.z, w.w};
                        const uint32_t at = index(static_cast<uint32_t>(q));
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e)
                        {
                            const uint64_t k = at + e < end && 4u * static_cast<uint32_t>(q) + e != taken ? make_key(f[e], at + e) : 0u;
                            const uint64_t all = __ballot(k > least);
                            if (k > least) queue[wave][waiting + __popcll(all & ((1ull << lane) - 1u))] = k;
                            waiting += static_cast<uint32_t>(__popcll(all));
                        }
                    }
                    __builtin_amdgcn_wave_barrier();
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    while (waiting >= 64u || (waiting >= enough && q + 1 == static_cast<int>(PER / 4u)))
                    {
                        const uint32_t n = min(waiting, 64u);
                        waiting -= n;
                        best = wave_merge(best, wave_sort(lane < n ? queue[wave][waiting + lane] : 0u));
                        least = key_at(best, p.top - 1u);
                        bar = least ? key_value(static_cast<uint32_t>(least >> 32)) : NEG_INF;
                    }
                }
            }
    }
    if constexpr (TOP)
    {
        __builtin_amdgcn_wave_barrier();
        queue[wave][lane] = best;
    }
    a = wave_stats(a, tau);
    if (lane == 0u) part[wave] = float4{a.m, a.s, a.e, a.bad ? 1.0f : 0.0f};
    __syncthreads();
    if (wave != 0u) return;
    const float4 mine = part[lane & 3u];
    a = wave_stats(Stats{lane < 4u ? mine.x : NEG_INF, lane < 4u ? mine.y : 0.0f, lane < 4u ? mine.z : 0.0f, lane < 4u && mine.w != 0.0f}, tau);
    if constexpr (TOP)
#pragma unroll 1
        for (uint32_t w = 1; w < 4; ++w) best = wave_merge(best, queue[w][63u - lane]);
    if constexpr (ONE) finish(p, row, a, best, Given(p, row));
    else
    {
        if (lane == 0u) p.stats[blockIdx.x] = float4{a.m, a.s, a.e, a.bad ? 1.0f : 0.0f};
        if (TOP && lane < p.top) p.keys[static_cast<uint64_t>(blockIdx.x) * p.top + lane] = best;
    }
}

// Joins a row's slices: each of W waves every W-th slice's keys, then four waves every
// fourth wave's, then one theirs.
template <bool TOP, uint32_t W>
__global__ __launch_bounds__(64 * W) void k_logprobs_join(LogprobParams p)
{
    constexpr uint32_t N = MAX_SLICES / 16u;             // slices a wave at most (W 16; W 4: up to 16 slices)
    __shared__ uint64_t list[W][64];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, row = blockIdx.x;
    const uint64_t at = static_cast<uint64_t>(row) * p.slices;
    const float4 mine = p.stats[at + min(lane, p.slices - 1u)];
    const Given given(p, row);
    uint64_t best = 0;
    if constexpr (TOP)
    {
        uint64_t k[N];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i)
        {
            const uint32_t s = wave + i * W, from = i ? 63u - lane : lane;
            k[i] = p.keys[(at + min(s, p.slices - 1u)) * p.top + min(from, p.top - 1u)];
            k[i] = s < p.slices && from < p.top ? k[i] : 0u;
        }
        best = k[0];
#pragma unroll
        for (uint32_t i = 1; i < N; ++i) best = wave_merge(best, k[i]);
        auto join = [&](uint32_t n, uint32_t by) {
            // wave w and w + by, w + 2 by, ... below n
#pragma unroll 1
            for (uint32_t w = wave + by; w < n; w += by) best = wave_merge(best, list[w][63u - lane]);
        };
        list[wave][lane] = best;
        __syncthreads();
        if constexpr (W > 4u)
        {
            if (wave < 4u)
            {
                join(min(W, p.slices), 4u);
                list[wave][lane] = best;
            }
            __syncthreads();
        }
        if (wave == 0u) join(4u, 1u);
    }
    if (wave != 0u) return;
    const bool in = lane < p.slices;
    finish(p, row, wave_stats(Stats{in ? mine.x : NEG_INF, in ? mine.y : 0.0f, in ? mine.z : 0.0f, in && mine.w != 0.0f}, p.temperature), best, given);
}

// A row in as many slices as give each CU four workgroups.
void slices_of(const opure_dev* dev, const opure_logprobs_args* a, uint32_t& slices, uint32_t& slice)
{
    const uint32_t cu = dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u, most = (a->vocab + 4u * CHUNK - 1u) / (4u * CHUNK);
    slices = std::min({std::max(1u, 4u * cu / a->rows), most, MAX_SLICES});
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
    if (!p.top) OPURE_LAUNCH(dev, (k_logprobs_join<false, 1>), dim3(p.rows), dim3(64), 0, p);
    else if (p.slices <= 16u) OPURE_LAUNCH(dev, (k_logprobs_join<true, 4>), dim3(p.rows), block, 0, p);
    else OPURE_LAUNCH(dev, (k_logprobs_join<true, 16>), dim3(p.rows), dim3(1024), 0, p);
    OPURE_LAUNCH_CHECK("k_logprobs_join");
    return OPURE_OK;
}
