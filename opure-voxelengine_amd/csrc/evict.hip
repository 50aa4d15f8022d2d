// ============================================================================
//  evict.hip -- eviction from the paged KV cache by accumulated attention
//  weight, in place, in place of the reference's EvictOldestKV and MemmoveMain
//  (Opure_VoxelEngine.cpp:721-763).
//
//  Of n positions of a (sequence, layer, KV head), keep = sinks + recent +
//  heavy: the first `sinks`, the last `recent`, and the `heavy` largest scores
//  between them.  With s_0 < s_1 < ... the kept positions, slot i takes V of s_i
//  and K of s_i, turned back by RoPE over s_i - i positions where asked.
//
//  In place: s_i >= i, so the slots that a run of kept positions moves to hold
//  no position that a later run still reads.
// ============================================================================
#include "internal.h"

#include <type_traits>

using namespace opure_dev_math;

namespace {

struct EvictParams {
    void* pool;
    int32_t* page_table;
    const int32_t* seq_len;
    const float* scores;
    float* scores_out;
    int32_t* kept;
    int32_t* new_len;
    int32_t* freed;
    int32_t* n_freed;
    const float* cos;
    const float* sin;
    uint32_t n_layers, n_kv, hd, n_pages, max_pages, afmt, scores_stride, sinks, recent, heavy, keep, freed_stride, cap;
    uint32_t new_len_now;         // no k_evict_finish follows: the selection writes the new lengths
    uint32_t* err;
};

__device__ __forceinline__ uint32_t evict_len(const EvictParams& p, uint32_t b)
{
    const int32_t n = p.seq_len[b];
    return n < 0 ? 0u : min(static_cast<uint32_t>(n), p.cap);
}

// a score as an unsigned number of the same order: NaN above +inf, -0 as +0
__device__ __forceinline__ uint32_t score_key(float f)
{
    if (f != f) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(f == 0.0f ? 0.0f : f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums over W waves in thread order of a count: those before this thread's, and all.
template <uint32_t W>
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* wsum, uint32_t& all)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (uint32_t o = 1; o < 64u; o <<= 1)
    {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63u) wsum[wave] = x;
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w)
    {
        const uint32_t s = wsum[w];
        before += w < wave ? s : 0u;
        all += s;
    }
    return before + x - v;
}

// The kept positions of one (sequence, layer, KV head), by 64 W threads.  First
// the `heavy`-th largest key, by counts of its leading 11, next 11 and last 10
// bits; then the positions above it and, from the lowest on, as many equal to it
// as are missing, in order.  A group that stays whole ends the counting.  A thread
// holds 4 consecutive scores in registers, so up to 256 W positions are read once,
// ordered by one prefix sum, and written with their scores as they are found (all
// scores are read by then: scores_out may be scores); longer sequences are read
// again, a block of 256 W at a time.  Bound by its chain of counts and barriers: a
// whole call of 128 small heads of 2,048 positions takes 20.8 us with 8 waves of 4
// scores a thread, 22.7 with 4 waves of 8 or 16 of 4.  More positions than a block
// and heads that leave CUs idle take 16 waves: 128 heads of 4,000 are 33.9 us, 38.5
// with 8, while 768 heads of 3,500 to 8,000 lose 6 us of 608 to them.
constexpr uint32_t SEL = 4;

template <uint32_t W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(W / 2))) void k_evict_select(EvictParams p)
{
    constexpr uint32_t T = 64u * W, BLOCK = T * SEL, BINS = 2048u, PER = BINS / T;
    __shared__ uint32_t hist[BINS], pick[3], wsum[4][W];
    const uint32_t b = blockIdx.y, tid = threadIdx.x;
    const uint64_t plane = static_cast<uint64_t>(b) * p.n_layers * p.n_kv + blockIdx.x;
    const int32_t raw = p.seq_len[b];
    const float* sc = p.scores + plane * p.scores_stride;
    const uint32_t n = raw < 0 ? 0u : min(static_cast<uint32_t>(raw), p.cap);
    int32_t* kept = p.kept + plane * p.keep;
    float* so = p.scores_out ? p.scores_out + plane * p.scores_stride : nullptr;
    const uint32_t lo = p.sinks, hi = n > p.keep ? n - p.recent : 0u;   // candidates lo .. hi - 1
    const uint32_t count = min(n, p.keep);
    const bool once = n <= BLOCK;
    if (tid == 0u && blockIdx.x == 0u)
    {
        if (raw < 0 || static_cast<uint32_t>(raw) > p.cap) p.err[ERR_POSITION] = 1u;
        if (p.new_len_now)
        {
            p.new_len[b] = static_cast<int32_t>(count);
            if (p.n_freed) p.n_freed[b] = 0;
        }
    }
    if (blockIdx.x == 0u)
    {
        // every page of the sequence, also those that the move has no need to read
        const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
        bool gone = false;
        for (uint32_t i = tid; i * OPURE_PAGE_SIZE < n; i += T) gone = gone || static_cast<uint32_t>(pt[i]) >= p.n_pages;
        if (gone) p.err[ERR_POSITION] = 1u;
    }
    if (n <= p.keep)
    {
        for (uint32_t i = tid; i < p.keep; i += T) kept[i] = i < n ? static_cast<int32_t>(i) : -1;
        if (so && so != sc)
            for (uint32_t i = tid; i < n; i += T) so[i] = sc[i];
        return;
    }
    float v[SEL];
    auto load = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t u = 0; u < SEL; ++u)
        {
            const uint32_t t = t0 + tid * SEL + u;
            v[u] = t < n ? sc[t] : 0.0f;
        }
    };
    load(0u);
    uint32_t prefix = 0, need = p.heavy;                   // the key's leading bits so far; how many still of its group
#pragma unroll
    for (uint32_t step = 0; step < 3u; ++step)
    {
        if (p.heavy == 0u) break;
        const uint32_t shift = step == 0u ? 21u : step == 1u ? 10u : 0u, bins = step == 2u ? 1024u : BINS;
        const uint32_t mask = step == 0u ? 0u : 0xFFFFFFFFu << (step == 1u ? 21u : 10u);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) hist[tid + T * i] = 0u;
        __syncthreads();
        for (uint32_t t0 = 0; t0 < hi; t0 += BLOCK)
        {
            if (!once) load(t0);
#pragma unroll
            for (uint32_t u = 0; u < SEL; ++u)
            {
                const uint32_t t = t0 + tid * SEL + u, key = score_key(v[u]);
                if (t >= lo && t < hi && (key & mask) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1u)], 1u);
            }
        }
        __syncthreads();
        // how many keys of the group lie above each of this thread's bins, from the top (the last step's upper bins are empty)
        uint32_t h[PER], sum = 0, all;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i)
        {
            h[i] = hist[BINS - 1u - (tid * PER + i)];
            sum += h[i];
        }
        uint32_t above = block_prefix<W>(sum, wsum[step], all);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i)
        {
            if (above < need && above + h[i] >= need)
            {
                pick[0] = BINS - 1u - (tid * PER + i);
                pick[1] = need - above;
                pick[2] = h[i];
            }
            above += h[i];
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        need = pick[1];
        if (step < 2u && need == pick[2])
        {
            // the whole group stays: all keys from its lowest on (no key is 0)
            --prefix;
            need = 0;
            break;
        }
    }
    uint32_t out = 0, equal = 0;                           // kept and equal keys of the blocks before
    for (uint32_t t0 = 0; t0 < n; t0 += BLOCK)
    {
        if (!once) load(t0);
        uint32_t sure = 0, eq = 0;                         // kept for certain; equal to the key
#pragma unroll
        for (uint32_t u = 0; u < SEL; ++u)
        {
            const uint32_t t = t0 + tid * SEL + u, key = score_key(v[u]);
            const bool cand = t >= lo && t < hi && p.heavy != 0u;
            sure += t < n && (t < lo || t >= hi || (cand && key > prefix)) ? 1u : 0u;
            eq += cand && key == prefix ? 1u : 0u;
        }
        // a block's counts stay below 2^16: both in one sum
        uint32_t all;
        if (!once) __syncthreads();                        // wsum of the block before is read
        const uint32_t at = block_prefix<W>(sure << 16 | eq, wsum[3], all);
        uint32_t eq_before = equal + (at & 0xFFFFu);
        uint32_t to = out + (at >> 16) + min(eq_before, need) - min(equal, need);
#pragma unroll
        for (uint32_t u = 0; u < SEL; ++u)
        {
            const uint32_t t = t0 + tid * SEL + u, key = score_key(v[u]);
            const bool cand = t >= lo && t < hi && p.heavy != 0u, same = cand && key == prefix;
            const bool stay = t < n && (t < lo || t >= hi || (cand && key > prefix) || (same && eq_before < need));
            eq_before += same ? 1u : 0u;
            if (stay)
            {
                kept[to] = static_cast<int32_t>(t);
                if (so && once) so[to] = v[u];
                ++to;
            }
        }
        const uint32_t eq_after = equal + (all & 0xFFFFu);
        out += (all >> 16) + min(eq_after, need) - min(equal, need);
        equal = eq_after;
    }
    if (!so) return;
    if (!once)
    {
        __syncthreads();                                   // the kept positions written, visible to the workgroup
        for (uint32_t i0 = 0; i0 < count; i0 += T)
        {
            const uint32_t i = i0 + tid;
            const float x = i < count ? sc[kept[i]] : 0.0f;
            __syncthreads();                               // scores_out may be scores: read before written
            if (i < count) so[i] = x;
        }
    }
    for (uint32_t i = count + tid; i < n; i += T) so[i] = 0.0f;
}

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// 16 bytes; ONCE: of a cache past the last-level cache, where nothing is met again before it is displaced
template <bool ONCE>
__device__ __forceinline__ u4v move_load(const uint8_t* p)
{
    const u4v* q = reinterpret_cast<const u4v*>(p);
    if constexpr (ONCE) return __builtin_nontemporal_load(q);
    else return *q;
}
template <bool ONCE>
__device__ __forceinline__ void move_store(uint8_t* p, u4v x)
{
    u4v* q = reinterpret_cast<u4v*>(p);
    if constexpr (ONCE) __builtin_nontemporal_store(x, q);
    else *q = x;
}

// a pair of a key's channels turned back by the angle of (c, s)
template <int AF>
__device__ __forceinline__ uint32_t turn_pair(uint32_t v, float c, float s)
{
    const float x = AF == OPURE_A_F16 ? f16_to_f32(static_cast<uint16_t>(v)) : bits_f(v << 16);
    const float y = AF == OPURE_A_F16 ? f16_to_f32(static_cast<uint16_t>(v >> 16)) : bits_f(v & 0xFFFF0000u);
    const float a = __fmaf_rn(x, c, __fmul_rn(y, s)), b = __fmaf_rn(y, c, -__fmul_rn(x, s));
    return AF == OPURE_A_F16 ? static_cast<uint32_t>(f32_to_f16(a)) | static_cast<uint32_t>(f32_to_f16(b)) << 16
                             : static_cast<uint32_t>(f32_to_bf16(a)) | static_cast<uint32_t>(f32_to_bf16(b)) << 16;
}

// Moves part of one (sequence, layer, KV head): 16 KP bytes of its K rows, or CH
// channels of its V planes, from the first position that can move to the last.
// Parts never meet, so all run at once; within one the runs go in order, a run's
// loads issued before the run before it is written (no slot that a run writes is
// read by a later one), with one barrier between a run's loads and its stores.
//   K: KP threads a position, 256 KU / KP kept positions a run, each thread's kept
// position, page and data fetched a run ahead of one another.
//   V: a channel's positions lie side by side, so runs of source pages go whole
// (their 32-byte rows hold a kept position nearly always) through LDS, rows of
// one channel, and the kept ones are collected from there into 16-byte stores;
// a group of positions that a run fills in part is stored by elements.
//   Bound by the cache's bytes: 32 layers of 3 sequences of 3,500 to 8,000
// positions cut to 2,504 (8 KV heads of 128) read K where it is kept, V whole and
// write both, 2.6 GB in 576 us, 4.5 TB/s (copies of 4 GiB reach 4.6 to 4.8, of 1 GiB
// 5.4); 16 layers of 2,048
// positions halved (heads of 64), 84 MB in 22 us.
//   KU: long runs keep more in flight a workgroup, short ones more workgroups a CU.
// Four where all workgroups fit at a time, three a CU (16 KV heads of 8,000 positions
// 61 us, 72 with one; the 16 layers 28.5, 29.7), else one (240 heads of 160 positions
// of 256 channels 33 -> 20 us, 256 heads of 1,000 of 128 53 -> 43).
//   A cache past the last-level cache (256 MB) moves K in whole 128-byte lines,
// which two parts on two XCDs would each fetch, and with accesses that do not stay
// in the caches: the 32 layers' call takes 790 us with 64-byte parts, 730 with lines,
// 668 streaming; 629 with V's channels by 32, a page's 1,024 bytes together (640
// with runs of twice the length, 730 with 64 channels), and 608 with KU 3 (1: 648, or
// 614 with 16 channels).  The 16 layers' takes 34 us with 64-byte parts, 39 with
// lines, 44 streaming.
template <int AF, uint32_t KP, uint32_t KU, uint32_t CH, bool ONCE>
__global__ __launch_bounds__(256) void k_evict_move(EvictParams p)
{
    constexpr uint32_t EB = AF == OPURE_A_F32 ? 4u : 2u, RUN = 1024u / EB, TPP = 16u / EB, PPC = 16u / TPP;
    constexpr uint32_t ROW = RUN * EB + 16u;               // bytes of a channel's row in LDS, a piece of padding
    __shared__ __align__(16) uint8_t rows[CH * ROW];
    __shared__ __align__(16) uint16_t from[RUN + 16u];     // the run's kept positions, from the run's first
    __shared__ uint32_t cnt[4];
    const uint32_t hd = p.hd, segk = (hd * EB + 16u * KP - 1u) / (16u * KP), segs = segk + hd / CH;
    const uint32_t b = blockIdx.y, head = blockIdx.x / segs, layer = head / p.n_kv, kh = head - layer * p.n_kv, tid = threadIdx.x;
    uint32_t seg = blockIdx.x - head * segs;
    const uint32_t n = evict_len(p, b);
    if (n <= p.keep) return;                               // every position stays where it is
    const int32_t* kept = p.kept + (static_cast<uint64_t>(b) * p.n_layers * p.n_kv + head) * p.keep;
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    const uint64_t plane = static_cast<uint64_t>(OPURE_PAGE_SIZE) * hd * EB, page_bytes = 2ull * p.n_kv * plane;
    uint8_t* base = static_cast<uint8_t*>(p.pool) + static_cast<uint64_t>(layer) * p.n_pages * page_bytes + kh * plane;
    auto there = [&](int32_t pg) { return static_cast<uint32_t>(pg) < p.n_pages; };
    if (seg < segk)
    {
        constexpr uint32_t U = KU, PASS = 256u / KP, KRUN = U * PASS;   // positions a pass; a run
        const uint32_t piece = seg * KP + tid % KP, tok = tid / KP;
        const bool mine = piece * 16u < hd * EB;
        const bool turn = p.cos != nullptr;
        auto kept_at = [&](uint32_t i) { return i < p.keep ? kept[i] : -1; };
        // (source position or -1, its page, the slot's page) of this thread's positions of a run
        int32_t s0[U], s1[U], ps[U], pd[U], qs[U], qd[U];
        u4v data[U], next[U];
        f4_t co[U], si[U], nco[U], nsi[U];
        const uint32_t first = p.sinks / KRUN * KRUN;
        auto pages = [&](uint32_t i0, const int32_t (&s)[U], int32_t (&a)[U], int32_t (&d)[U]) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
            {
                const uint32_t i = i0 + PASS * u + tok;
                const bool moves = mine && s[u] > static_cast<int32_t>(i);
                a[u] = moves ? pt[static_cast<uint32_t>(s[u]) / OPURE_PAGE_SIZE] : -1;
                d[u] = moves ? pt[i / OPURE_PAGE_SIZE] : -1;
                if (moves && !(there(a[u]) && there(d[u])))
                {
                    p.err[ERR_POSITION] = 1u;
                    a[u] = d[u] = -1;
                }
            }
        };
        auto load = [&](uint32_t i0, const int32_t (&s)[U], const int32_t (&a)[U], u4v (&x)[U], f4_t (&c)[U], f4_t (&sn)[U]) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
            {
                const uint32_t i = i0 + PASS * u + tok;
                if (a[u] < 0) continue;
                const uint32_t t = static_cast<uint32_t>(s[u]);
                x[u] = move_load<ONCE>(base + static_cast<uint32_t>(a[u]) * page_bytes + (t % OPURE_PAGE_SIZE) * (hd * EB) + piece * 16u);
                if (turn)
                {
                    const uint64_t at = static_cast<uint64_t>(t - i) * (hd / 2u) + piece * (TPP / 2u);
                    if constexpr (AF == OPURE_A_F32)
                    {
                        c[u][0] = p.cos[at], c[u][1] = p.cos[at + 1u];
                        sn[u][0] = p.sin[at], sn[u][1] = p.sin[at + 1u];
                    }
                    else
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)
                        {
                            c[u][k] = p.cos[at + k];
                            sn[u][k] = p.sin[at + k];
                        }
                }
            }
        };
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
        {
            s0[u] = kept_at(first + PASS * u + tok);
            s1[u] = kept_at(first + KRUN + PASS * u + tok);
        }
        pages(first, s0, ps, pd);
        load(first, s0, ps, data, co, si);
        pages(first + KRUN, s1, qs, qd);
        for (uint32_t i0 = first; i0 < p.keep; i0 += KRUN)
        {
            int32_t s2[U], rs[U], rd[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) s2[u] = kept_at(i0 + 2u * KRUN + PASS * u + tok);
            load(i0 + KRUN, s1, qs, next, nco, nsi);
            __syncthreads();
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
            {
                if (ps[u] < 0) continue;
                const uint32_t i = i0 + PASS * u + tok;
                u4v x = data[u];
                if (turn)
                {
                    if constexpr (AF == OPURE_A_F32)
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k)
                        {
                            const float a = bits_f(x[2 * k]), c = bits_f(x[2 * k + 1]);
                            x[2 * k] = f_bits(__fmaf_rn(a, co[u][k], __fmul_rn(c, si[u][k])));
                            x[2 * k + 1] = f_bits(__fmaf_rn(c, co[u][k], -__fmul_rn(a, si[u][k])));
                        }
                    else
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) x[k] = turn_pair<AF>(x[k], co[u][k], si[u][k]);
                }
                move_store<ONCE>(base + static_cast<uint32_t>(pd[u]) * page_bytes + (i % OPURE_PAGE_SIZE) * (hd * EB) + piece * 16u, x);
            }
            pages(i0 + 2u * KRUN, s2, rs, rd);
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
            {
                s0[u] = s1[u];
                s1[u] = s2[u];
                ps[u] = qs[u];
                pd[u] = qd[u];
                qs[u] = rs[u];
                qd[u] = rd[u];
                data[u] = next[u];
                co[u] = nco[u];
                si[u] = nsi[u];
            }
        }
        return;
    }
    // ---- V: CH channels
    seg -= segk;
    constexpr uint32_t U = CH / 4u, PG = RUN / OPURE_PAGE_SIZE, PPP = CH * PPC;   // pages a run; pieces a page
    static_assert(PG * PPP == 256u * U, "a run is U pieces a thread");
    uint8_t* vbase = base + p.n_kv * plane + static_cast<uint64_t>(seg) * CH * OPURE_PAGE_SIZE * EB;
    const uint32_t wave = tid >> 6, lane = tid & 63u;
    u4v data[U];
    int32_t pe[U];
    auto entries = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
        {
            const uint32_t t = t0 + (u * 256u + tid) / PPP * OPURE_PAGE_SIZE;
            pe[u] = t < n ? pt[t / OPURE_PAGE_SIZE] : -1;
            if (t < n && !there(pe[u]))
            {
                p.err[ERR_POSITION] = 1u;
                pe[u] = -1;
            }
        }
    };
    auto load = [&] {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            if (pe[u] >= 0)
                data[u] = move_load<ONCE>(vbase + static_cast<uint32_t>(pe[u]) * page_bytes + (u * 256u + tid) % PPP * 16u);
    };
    constexpr uint32_t KW = RUN / 256u;
    int32_t kw[KW];
    uint32_t t0 = p.sinks / RUN * RUN, i0 = t0;            // everything before the sinks' end stays in place
    auto window = [&](uint32_t i) {
#pragma unroll
        for (uint32_t k = 0; k < KW; ++k) kw[k] = i + 256u * k + tid < p.keep ? kept[i + 256u * k + tid] : 0x7FFFFFFF;
    };
    window(i0);
    entries(t0);
    load();
    entries(t0 + RUN);
    for (; i0 < p.keep && t0 < n; t0 += RUN)
    {
        __syncthreads();                                   // the run before is collected
        uint32_t c = 0;
        const uint32_t d0 = i0 / OPURE_PAGE_SIZE;
#pragma unroll
        for (uint32_t k = 0; k < KW; ++k)
        {
            const bool in = static_cast<uint32_t>(kw[k]) < t0 + RUN;
            c += static_cast<uint32_t>(__popcll(__ballot(in)));
            if (in) from[i0 - d0 * OPURE_PAGE_SIZE + 256u * k + tid] = static_cast<uint16_t>(static_cast<uint32_t>(kw[k]) - t0);
        }
        if (lane == 0u) cnt[wave] = c;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
        {
            const uint32_t e = u * 256u + tid, pg = e / PPP, ch = e % PPP / PPC, half = e % PPC;
            *reinterpret_cast<u4v*>(rows + ch * ROW + (pg * PPC + half) * 16u) = data[u];
        }
        __syncthreads();
        const uint32_t i1 = i0 + cnt[0] + cnt[1] + cnt[2] + cnt[3];
        window(i1);
        load();
        entries(t0 + 2u * RUN);
        if (i1 > i0)
        {
            const uint32_t d1 = (i1 - 1u) / OPURE_PAGE_SIZE;
            for (uint32_t e = tid; e < (d1 - d0 + 1u) * PPP; e += 256u)
            {
                const uint32_t pg = d0 + e / PPP, ch = e % PPP / PPC, half = e % PPC, g0 = pg * OPURE_PAGE_SIZE + half * TPP;
                const uint32_t a = max(g0, i0), z = min(g0 + TPP, i1);
                if (a >= z) continue;
                const uint16_t* f = from + (g0 - d0 * OPURE_PAGE_SIZE);
                if (t0 + f[z - 1u - g0] == z - 1u) continue;   // the last one does not move, so none does
                const int32_t to = pt[pg];
                if (!there(to)) continue;                      // reported by the runs that read it
                uint8_t* dst = vbase + static_cast<uint32_t>(to) * page_bytes + (ch * PPC + half) * 16u;
                const uint8_t* row = rows + ch * ROW;
                if (z - a == TPP)
                {
                    u4v x;
                    if constexpr (EB == 4u)
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const uint32_t*>(row + f[k] * 4u);
                    else
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)
                            x[k] = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + f[2 * k] * 2u)) |
                                   static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + f[2 * k + 1] * 2u)) << 16;
                    move_store<ONCE>(dst, x);
                }
                else
                    for (uint32_t i = a; i < z; ++i)
                    {
                        if constexpr (EB == 4u) reinterpret_cast<uint32_t*>(dst)[i - g0] = *reinterpret_cast<const uint32_t*>(row + f[i - g0] * 4u);
                        else reinterpret_cast<uint16_t*>(dst)[i - g0] = *reinterpret_cast<const uint16_t*>(row + f[i - g0] * 2u);
                    }
            }
        }
        i0 = i1;
    }
}

// New lengths and, with `freed`, the pages past them: a wave a sequence.
__global__ __launch_bounds__(64) void k_evict_finish(EvictParams p)
{
    const uint32_t b = blockIdx.x, lane = threadIdx.x, n = evict_len(p, b), nl = min(n, p.keep);
    int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    uint32_t nf = 0;
    if (p.freed)
        for (uint32_t q0 = (nl + OPURE_PAGE_SIZE - 1u) / OPURE_PAGE_SIZE; q0 * OPURE_PAGE_SIZE < n; q0 += 64u)
        {
            const uint32_t q = q0 + lane;
            const int32_t pg = q * OPURE_PAGE_SIZE < n ? pt[q] : -1;
            const uint64_t has = __ballot(pg >= 0);
            if (pg >= 0)
            {
                p.freed[static_cast<uint64_t>(b) * p.freed_stride + nf + __popcll(has & ((1ull << lane) - 1u))] = pg;
                pt[q] = -1;
            }
            nf += static_cast<uint32_t>(__popcll(has));
        }
    if (lane == 0u)
    {
        p.new_len[b] = static_cast<int32_t>(nl);
        if (p.n_freed) p.n_freed[b] = static_cast<int32_t>(nf);
    }
}

}  // namespace

using namespace opure_hip;

namespace {

// What the call writes lies apart from everything else that it takes, but for
// scores_out at scores and new_seq_len at seq_len.
int evict_apart(const opure_evict_args* a, uint64_t keep)
{
    const opure_model* m = a->model;
    const opure_kv* kv = a->kv;
    const uint64_t planes = static_cast<uint64_t>(m->n_layers) * m->n_kv_heads, rows = a->batch * planes;
    const uint64_t scores = ((rows - 1u) * a->scores_stride + a->max_ctx) * 4u, lens = a->batch * 4u;
    const uint64_t freed = (static_cast<uint64_t>(a->batch - 1u) * a->freed_stride + (a->max_ctx + OPURE_PAGE_SIZE - 1u) / OPURE_PAGE_SIZE) * 4u;
    enum { POOL, TABLE, KEPT, SCORES, SCORES_OUT, LEN, NEW_LEN, FREED, N_FREED, PARTS };
    const struct { const char* name; const void* at; uint64_t bytes; bool written; } part[PARTS] = {
        {"pool", kv->pool, planes * kv->n_pages * 2u * OPURE_PAGE_SIZE * m->head_dim * act_bytes(m->afmt), true},
        {"page_table", kv->page_table, static_cast<uint64_t>(a->batch) * kv->max_pages_per_seq * 4u, a->freed != nullptr},
        {"kept", a->kept, rows * keep * 4u, true},
        {"scores", a->scores, scores, false},
        {"scores_out", a->scores_out, scores, true},
        {"seq_len", a->seq_len, lens, false},
        {"new_seq_len", a->new_seq_len, lens, true},
        {"freed", a->freed, freed, true},
        {"n_freed", a->n_freed, lens, true}};
    // scores_out between the rows of scores: the nearest two decide
    const int64_t d = a->scores_out ? a->scores_out - a->scores : 0, stride = a->scores_stride, last = static_cast<int64_t>(rows) - 1;
    bool meet = false;
    for (int64_t k = -(d / stride) - 1; k <= -(d / stride) + 1; ++k)
        meet = meet || (k >= -last && k <= last && d + k * stride < a->max_ctx && d + k * stride > -static_cast<int64_t>(a->max_ctx));
    for (int x = 0; x < PARTS; ++x)
        for (int y = x + 1; y < PARTS; ++y)
        {
            if (!(part[x].written || part[y].written) || !overlaps(part[x].at, part[x].bytes, part[y].at, part[y].bytes)) continue;
            if (x == SCORES && y == SCORES_OUT && (d == 0 || !meet)) continue;
            if (x == LEN && y == NEW_LEN && part[x].at == part[y].at) continue;
            return set_error(OPURE_E_INVALID, "opure_kv_evict: %s overlaps %s", part[y].name, part[x].name);
        }
    return OPURE_OK;
}

}  // namespace

extern "C" int opure_kv_evict(opure_dev* dev, const opure_evict_args* a)
{
    OPURE_REQUIRE(dev && a && a->model && a->kv && a->kv->pool && a->kv->page_table && a->seq_len && a->scores && a->kept &&
                      a->new_seq_len, OPURE_E_INVALID, "opure_kv_evict: null argument");
    const opure_model* m = a->model;
    const opure_kv* kv = a->kv;
    OPURE_REQUIRE(m->n_layers >= 1 && m->n_kv_heads >= 1 && m->afmt <= OPURE_A_BF16, OPURE_E_INVALID, "opure_kv_evict: bad model");
    OPURE_REQUIRE(m->head_dim >= 16 && m->head_dim <= 256 && m->head_dim % 16 == 0, OPURE_E_UNSUPPORTED,
                  "opure_kv_evict: head_dim %u not in 16..256 step 16", m->head_dim);
    OPURE_REQUIRE(kv->page_size == OPURE_PAGE_SIZE, OPURE_E_UNSUPPORTED, "opure_kv_evict: page_size must be %d", OPURE_PAGE_SIZE);
    OPURE_REQUIRE(kv->n_pages >= 1 && kv->max_pages_per_seq >= 1, OPURE_E_INVALID, "opure_kv_evict: the cache has no pages");
    OPURE_REQUIRE(a->batch >= 1 && a->batch <= OPURE_MAX_BATCH_ROWS, OPURE_E_CAPACITY, "opure_kv_evict: %u sequences outside 1..%d",
                  a->batch, OPURE_MAX_BATCH_ROWS);
    OPURE_REQUIRE(static_cast<uint64_t>(m->n_layers) * m->n_kv_heads <= 0x7FFFFu, OPURE_E_CAPACITY, "opure_kv_evict: %u layers x %u KV heads",
                  m->n_layers, m->n_kv_heads);
    const uint64_t slots = static_cast<uint64_t>(kv->max_pages_per_seq) * OPURE_PAGE_SIZE;
    OPURE_REQUIRE(a->max_ctx >= 1 && a->max_ctx <= slots && a->max_ctx <= 0x7FFFFFFFu, OPURE_E_CAPACITY,
                  "opure_kv_evict: max_ctx %u beyond the page table's %llu", a->max_ctx, (unsigned long long)slots);
    OPURE_REQUIRE(a->scores_stride >= a->max_ctx, OPURE_E_INVALID, "opure_kv_evict: scores_stride %u below max_ctx %u",
                  a->scores_stride, a->max_ctx);
    const uint64_t keep = static_cast<uint64_t>(a->sinks) + a->recent + a->heavy;
    OPURE_REQUIRE(keep >= 1 && keep <= 0x7FFFFFFFu, OPURE_E_INVALID, "opure_kv_evict: %llu positions to keep", (unsigned long long)keep);
    OPURE_REQUIRE(!a->turn || (m->rope_cos && m->rope_sin && m->rope_max_pos >= a->max_ctx), OPURE_E_INVALID,
                  "opure_kv_evict: turning keys needs RoPE tables of max_ctx %u positions", a->max_ctx);
    OPURE_REQUIRE(!a->freed || a->freed_stride >= (a->max_ctx + OPURE_PAGE_SIZE - 1u) / OPURE_PAGE_SIZE, OPURE_E_INVALID,
                  "opure_kv_evict: freed_stride %u below the pages of max_ctx %u", a->freed_stride, a->max_ctx);
    OPURE_REQUIRE((reinterpret_cast<uintptr_t>(kv->pool) & 15u) == 0u, OPURE_E_INVALID, "opure_kv_evict: pool must be 16-byte aligned");
    OPURE_REQUIRE(((reinterpret_cast<uintptr_t>(a->scores) | reinterpret_cast<uintptr_t>(a->scores_out) | reinterpret_cast<uintptr_t>(a->kept) |
                    reinterpret_cast<uintptr_t>(a->seq_len) | reinterpret_cast<uintptr_t>(a->new_seq_len) | reinterpret_cast<uintptr_t>(a->freed) |
                    reinterpret_cast<uintptr_t>(a->n_freed) | reinterpret_cast<uintptr_t>(kv->page_table)) & 3u) == 0u, OPURE_E_INVALID,
                  "opure_kv_evict: scores, kept, lengths and tables must be 4-byte aligned");
    const int rc = evict_apart(a, keep);
    if (rc) return rc;
    const DeviceGuard on(dev);
    EvictParams p{};
    p.pool = kv->pool;
    p.page_table = kv->page_table;
    p.seq_len = a->seq_len;
    p.scores = a->scores;
    p.scores_out = a->scores_out;
    p.kept = a->kept;
    p.new_len = a->new_seq_len;
    p.freed = a->freed;
    p.n_freed = a->n_freed;
    p.cos = a->turn ? m->rope_cos : nullptr;
    p.sin = a->turn ? m->rope_sin : nullptr;
    p.n_layers = m->n_layers;
    p.n_kv = m->n_kv_heads;
    p.hd = m->head_dim;
    p.n_pages = kv->n_pages;
    p.max_pages = kv->max_pages_per_seq;
    p.afmt = m->afmt;
    p.scores_stride = a->scores_stride;
    p.sinks = a->sinks;
    p.recent = a->recent;
    p.heavy = a->heavy;
    p.keep = static_cast<uint32_t>(keep);
    p.freed_stride = a->freed_stride;
    p.cap = a->max_ctx;
    p.err = dev->err;
    // the other workgroups read seq_len and the table: what is written over them waits for a launch of its own
    p.new_len_now = !a->freed && a->new_seq_len != a->seq_len ? 1u : 0u;
    const uint32_t planes = p.n_layers * p.n_kv;
    if (a->max_ctx <= 8u * 64u * SEL || planes * a->batch > 256u) OPURE_LAUNCH(dev, (k_evict_select<8>), dim3(planes, a->batch), dim3(512), 0, p);
    else OPURE_LAUNCH(dev, (k_evict_select<16>), dim3(planes, a->batch), dim3(1024), 0, p);
    OPURE_LAUNCH_CHECK("k_evict_select");
    const uint32_t row = p.hd * act_bytes(p.afmt);
    const bool once = static_cast<uint64_t>(planes) * a->batch * a->max_ctx * row * 2u > 256u << 20;
    auto move = [&](auto af) {
        constexpr int AF = decltype(af)::value;
        auto go = [&](auto kernel, uint32_t kp, uint32_t ch) {
            OPURE_LAUNCH(dev, kernel, dim3(planes * ((row + 16u * kp - 1u) / (16u * kp) + p.hd / ch), a->batch), dim3(256), 0, p);
        };
        const uint64_t wgs = static_cast<uint64_t>(planes) * ((row + 63u) / 64u + p.hd / 16u) * a->batch;
        if (!once && wgs <= 3u * static_cast<uint32_t>(dev->n_cu > 0 ? dev->n_cu : 256)) go(&k_evict_move<AF, 4, 4, 16, false>, 4u, 16u);
        else if (!once) go(&k_evict_move<AF, 4, 1, 16, false>, 4u, 16u);
        else if (row % 128u == 0u) go(&k_evict_move<AF, 8, 3, 32, true>, 8u, 32u);
        else go(&k_evict_move<AF, 4, 1, 16, true>, 4u, 16u);
    };
    if (p.afmt == OPURE_A_F32) move(std::integral_constant<int, OPURE_A_F32>{});
    else if (p.afmt == OPURE_A_F16) move(std::integral_constant<int, OPURE_A_F16>{});
    else move(std::integral_constant<int, OPURE_A_BF16>{});
    OPURE_LAUNCH_CHECK("k_evict_move");
    if (p.new_len_now) return OPURE_OK;
    OPURE_LAUNCH(dev, k_evict_finish, dim3(a->batch), dim3(64), 0, p);
    OPURE_LAUNCH_CHECK("k_evict_finish");
    return OPURE_OK;
}
