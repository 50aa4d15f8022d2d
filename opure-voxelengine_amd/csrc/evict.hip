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

// Sums over 1,024 threads in thread order: the sum of those before this one,
// and of all.
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
    __syncthreads();                                       // wsum of the call before is read
    if (lane == 63u) wsum[wave] = x;
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < 16u; ++w)
    {
        const uint32_t s = wsum[w];
        before += w < wave ? s : 0u;
        all += s;
    }
    return before + x - v;
}

// The kept positions of one (sequence, layer, KV head): the `heavy`-th largest
// key by four counts of 8 bits each, then the positions above it and, from the
// lowest on, as many equal to it as are missing, written in order.
__global__ __launch_bounds__(1024) void k_evict_select(EvictParams p)
{
    __shared__ uint32_t hist[256], wsum[16], pick[2];
    const uint32_t b = blockIdx.y, tid = threadIdx.x;
    const uint64_t plane = static_cast<uint64_t>(b) * p.n_layers * p.n_kv + blockIdx.x;
    const int32_t raw = p.seq_len[b];
    const uint32_t n = evict_len(p, b);
    if (tid == 0u && blockIdx.x == 0u && (raw < 0 || static_cast<uint32_t>(raw) > p.cap)) p.err[ERR_POSITION] = 1u;
    const float* sc = p.scores + plane * p.scores_stride;
    int32_t* kept = p.kept + plane * p.keep;
    const uint32_t lo = p.sinks, hi = n > p.keep ? n - p.recent : 0u;   // candidates lo .. hi - 1
    const uint32_t count = min(n, p.keep);
    if (n <= p.keep)
    {
        for (uint32_t i = tid; i < p.keep; i += 1024u) kept[i] = i < n ? static_cast<int32_t>(i) : -1;
    }
    else
    {
        uint32_t prefix = 0, need = p.heavy;               // the key's leading bits so far; how many still of its group
        if (p.heavy)
            for (int shift = 24; shift >= 0; shift -= 8)
            {
                if (tid < 256u) hist[tid] = 0u;
                __syncthreads();
                const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
                for (uint32_t t = lo + tid; t < hi; t += 1024u)
                {
                    const uint32_t k = score_key(sc[t]);
                    if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
                }
                __syncthreads();
                // how many keys of the group lie above each bin, from the top
                uint32_t all;
                const uint32_t h = tid < 256u ? hist[255u - tid] : 0u;
                const uint32_t above = block_prefix(h, wsum, all);
                if (tid < 256u && above < need && above + h >= need)
                {
                    pick[0] = 255u - tid;
                    pick[1] = need - above;
                }
                __syncthreads();
                prefix |= pick[0] << shift;
                need = pick[1];
                __syncthreads();
            }
        uint32_t out = 0, equal = 0;                       // kept so far; equal keys so far
        for (uint32_t t0 = 0; t0 < n; t0 += 1024u)
        {
            const uint32_t t = t0 + tid;
            const bool fixed = t < n && (t < lo || t >= hi);
            const uint32_t k = t >= lo && t < hi ? score_key(sc[t]) : 0u;
            const bool cand = t >= lo && t < hi && p.heavy != 0u, eq = cand && k == prefix;
            uint32_t all_eq, all;
            const uint32_t eq_before = block_prefix(eq ? 1u : 0u, wsum, all_eq);
            const bool stay = fixed || (cand && k > prefix) || (eq && equal + eq_before < need);
            const uint32_t at = block_prefix(stay ? 1u : 0u, wsum, all);
            if (stay) kept[out + at] = static_cast<int32_t>(t);
            out += all;
            equal += all_eq;
        }
    }
    if (p.scores_out)
    {
        float* so = p.scores_out + plane * p.scores_stride;
        __syncthreads();                                   // the kept positions written, visible to the workgroup
        for (uint32_t i0 = 0; i0 < count; i0 += 1024u)
        {
            const uint32_t i = i0 + tid;
            const float v = i < count ? sc[kept[i]] : 0.0f;
            __syncthreads();                               // scores_out may be scores: read before written
            if (i < count) so[i] = v;
        }
        __syncthreads();
        for (uint32_t i = count + tid; i < n; i += 1024u) so[i] = 0.0f;
    }
}

// Moves the K (y = 0) or V (y = 1) plane of one (sequence, layer, KV head): a
// run of 16 kept positions at a time, all of them read before any is written.
__global__ __launch_bounds__(256) void k_evict_move(EvictParams p)
{
    const uint32_t b = blockIdx.z, layer = blockIdx.x / p.n_kv, kh = blockIdx.x - layer * p.n_kv, which = blockIdx.y;
    const uint32_t n = evict_len(p, b), tid = threadIdx.x, hd = p.hd;
    if (n <= p.keep) return;                               // every position stays where it is
    const int32_t* kept = p.kept + (static_cast<uint64_t>(b) * p.n_layers * p.n_kv + blockIdx.x) * p.keep;
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    auto page = [&](uint32_t t) -> int32_t {
        const int32_t pg = pt[t / OPURE_PAGE_SIZE];
        if (pg >= 0 && static_cast<uint32_t>(pg) < p.n_pages) return pg;
        p.err[ERR_POSITION] = 1u;
        return -1;
    };
    for (uint32_t i0 = 0; i0 < p.keep; i0 += OPURE_PAGE_SIZE)
    {
        // 16 positions x hd channels: up to 8 pairs of channels a thread
        float x[8], y[8];
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u)
        {
            const uint32_t e = tid + 256u * u, i = i0 + e % OPURE_PAGE_SIZE, c = e / OPURE_PAGE_SIZE;
            x[u] = y[u] = 0.0f;
            if (2u * c >= hd || i >= p.keep) continue;
            const uint32_t s = static_cast<uint32_t>(kept[i]);
            const int32_t pg = page(s);
            if (pg < 0) continue;
            const uint32_t d = 2u * c;
            float k0 = load_act_rt(p.pool, kv_elem(layer, p.n_pages, pg, which, p.n_kv, kh, hd, s % OPURE_PAGE_SIZE, d), p.afmt);
            float k1 = load_act_rt(p.pool, kv_elem(layer, p.n_pages, pg, which, p.n_kv, kh, hd, s % OPURE_PAGE_SIZE, d + 1u), p.afmt);
            if (which == 0u && p.cos && s != i)
            {
                const float co = p.cos[static_cast<uint64_t>(s - i) * (hd / 2u) + c], si = p.sin[static_cast<uint64_t>(s - i) * (hd / 2u) + c];
                const float r0 = __fmaf_rn(k0, co, __fmul_rn(k1, si)), r1 = __fmaf_rn(k1, co, -__fmul_rn(k0, si));
                k0 = r0;
                k1 = r1;
            }
            x[u] = k0;
            y[u] = k1;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u)
        {
            const uint32_t e = tid + 256u * u, i = i0 + e % OPURE_PAGE_SIZE, c = e / OPURE_PAGE_SIZE;
            if (2u * c >= hd || i >= p.keep || static_cast<uint32_t>(kept[i]) == i) continue;
            const int32_t pg = page(i);
            if (pg < 0) continue;
            const uint32_t d = 2u * c;
            store_act_rt(p.pool, kv_elem(layer, p.n_pages, pg, which, p.n_kv, kh, hd, i % OPURE_PAGE_SIZE, d), x[u], p.afmt);
            store_act_rt(p.pool, kv_elem(layer, p.n_pages, pg, which, p.n_kv, kh, hd, i % OPURE_PAGE_SIZE, d + 1u), y[u], p.afmt);
        }
        __syncthreads();
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
    OPURE_REQUIRE(static_cast<uint64_t>(m->n_layers) * m->n_kv_heads <= 0x7FFFFFu, OPURE_E_CAPACITY, "opure_kv_evict: %u layers x %u KV heads",
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
    const uint32_t planes = p.n_layers * p.n_kv;
    OPURE_LAUNCH(dev, k_evict_select, dim3(planes, a->batch), dim3(1024), 0, p);
    OPURE_LAUNCH_CHECK("k_evict_select");
    OPURE_LAUNCH(dev, k_evict_move, dim3(planes, 2, a->batch), dim3(256), 0, p);
    OPURE_LAUNCH_CHECK("k_evict_move");
    OPURE_LAUNCH(dev, k_evict_finish, dim3(a->batch), dim3(64), 0, p);
    OPURE_LAUNCH_CHECK("k_evict_finish");
    return OPURE_OK;
}
