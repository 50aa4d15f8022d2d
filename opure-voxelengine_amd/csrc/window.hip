// ============================================================================
//  window.hip -- attention over the paged cache with a sliding window and a few
//  first positions that stay visible, and the accumulated weights of the cached
//  positions that an eviction goes by.
//
//  Row j of a sequence, at position p = seq_len + j, sees t <= p with t < sinks
//  or t > p - window:  s_t = scale q.k_t,  w_t = exp(s_t - m) / sum exp(s - m),
//  out = sum w_t v_t, and weights[h][t] += w_t over the rows and the query heads
//  of KV head h.
// ============================================================================
#include "window.h"

#include <algorithm>
#include <cmath>

using namespace opure_win;
using opure_hip::act_bytes;

namespace {

constexpr uint32_t MAX_PARTS = 64;                         // of a (sequence, KV head, block of query rows): a lane of the joining wave each

// Few query rows: a workgroup takes a part of the tiles that a sequence's rows
// see, for 16 NT query rows of a KV head (row qi = j group + head), a wave every
// fourth tile with a running maximum, sum and output of its own in registers.
// Bound by the cache's bytes.  A tile's K goes to the matrix unit and the next
// one's loads into the same registers at once, its V likewise, so a wave has
// about a tile (16 KB at 128 channels) in flight all the time without a second
// set of registers.  The four waves are merged in LDS, the parts by k_win_join.
//   A probability enters its product as two 16-bit numbers (its rounding and the
// rest: 16 bits in bf16, so that 2^-16 of it is lost where the result's own rounding
// is 2^-8, and 22 in fp16, against 2^-11): the products are not what bounds this.
//   ONCE: at most 16 query rows a KV head, so no other workgroup reads its bytes, and
// the loads stream.  Past 128 channels more rows are more blocks of 16, which find
// each other's bytes in the caches (streaming / not: 16 rows of 64 heads of 256 over
// 8,000 positions 88.0 / 58.9 us, 12 of 16 heads of 160 in 8 sequences of 4,000 46.5 /
// 32.2, an fp32 prompt of 2,048 rows of 4 heads of 256 231 / 211).
//   32 sequences of 1,024 to 16,384 positions behind a window of 4,096 (8 KV heads
// of 128) read 412 MB in 75 us, 5.5 TB/s; reads alone of scattered 2 KB planes reach
// 5.8.  One row over 1,000 positions of heads of 64 takes 4.4 us, a chain of
// round trips (length, page entries, keys and values) rather than bytes.
template <int AF, int HD, int NT, bool ONCE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NT == 2 ? 2 : 1))) void k_win_split(WinParams p)
{
    typedef WinTile<AF, HD> T;
    constexpr uint32_t TT = T::TT, DT = T::DT, NS = T::NS;
    extern __shared__ __align__(16) uint8_t lds[];
    f4_t* cacc = reinterpret_cast<f4_t*>(lds);                            // [wave][DT][NT][64]
    float* cml = reinterpret_cast<float*>(lds + 4u * DT * NT * 64u * 16u);   // [wave][NT][16][2]
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t G = p.n_heads / p.n_kv, Gq = G * p.rows;
    // KV heads next to each other, then parts, blocks and sequences
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, part = rest % p.parts;
    const uint32_t b = rest / p.parts / p.blocks, blk = rest / p.parts - b * p.blocks, q0 = blk * 16u * NT;
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    const int32_t len = p.seq_len[b];
    u4v q[NT][T::KS];
    uint32_t jr[NT];
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
    {
        const uint32_t qi = min(q0 + 16u * n + r, Gq - 1u);
        jr[n] = qi / G;
        win_load_q<AF, HD>(p, (static_cast<uint64_t>(b) * p.rows + jr[n]) * p.n_heads + kh * G + (qi - jr[n] * G), g, q[n]);
    }
    const WinSeq sq = win_seq(p, len);
    // the list is the whole sequence's, so that a tile has one place among the scores whatever the block
    const WinSpan span = win_span<TT>(p, sq, sq.ctx, sq.ctx + p.rows);
    const uint32_t j0 = q0 / G, j1 = min(q0 + 16u * NT - 1u, Gq - 1u) / G;    // the block's first and last row
    const uint32_t first = static_cast<uint32_t>(static_cast<uint64_t>(span.n) * part / p.parts);
    const uint32_t last = static_cast<uint32_t>(static_cast<uint64_t>(span.n) * (part + 1u) / p.parts);
    const float c = __fmul_rn(p.scale, 1.44269504088896340736f);
    const uint64_t page_bytes = 2ull * p.n_kv * T::PB;
    const uint8_t* kbase = static_cast<const uint8_t*>(p.pool) + static_cast<uint64_t>(p.layer) * p.n_pages * page_bytes + static_cast<uint64_t>(kh) * T::PB;
    const uint64_t vofs = static_cast<uint64_t>(p.n_kv) * T::PB;

    f4_t o[DT][NT];
    float m[NT], l[NT];
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
    {
        m[n] = NEG_INF;
        l[n] = 0.0f;
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d) o[d][n] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // pages of tile i of the list: -1 past the sequence, missing or not in the pool
    auto entry = [&](uint32_t i) { return pt[min(span.tile(min(i, span.n - 1u)) * T::NB + (lane & (T::NB - 1u)), p.max_pages - 1u)]; };
    auto page = [&](int32_t e, uint32_t i, uint32_t which) -> int32_t {
        const int32_t pg = __builtin_amdgcn_readlane(e, which);
        return (span.tile(i) * T::NB + which) * OPURE_PAGE_SIZE < sq.total && static_cast<uint32_t>(pg) < p.n_pages ? pg : -1;
    };
    T tl;
    uint32_t i = first + wave;
    if (i < last)
    {
        int32_t e = entry(i);
        int32_t pa = page(e, i, 0u), pb = T::NB > 1u ? page(e, i, 1u) : pa;
        auto at = [&](int32_t pg) { return kbase + static_cast<uint64_t>(pg < 0 ? 0u : static_cast<uint32_t>(pg)) * page_bytes; };
        tl.template load_k<ONCE>(at(pa), at(pb), r, g);
        tl.template load_v<ONCE>(at(pa) + vofs, at(pb) + vofs, r, g);
        e = entry(i + 4u);
        while (true)
        {
            const uint32_t t0 = span.tile(i) * TT;
            const bool more = i + 4u < last;
            const int32_t na = more ? page(e, i + 4u, 0u) : pa, nb = T::NB > 1u ? (more ? page(e, i + 4u, 1u) : pb) : na;
            if (more) e = entry(i + 8u);
            if (pa < 0 || pb < 0)
            {
                // positions without a page: NaN keys for the rows that see them, no values
                const uint32_t nan = AF == OPURE_A_F32 ? 0x7FC00000u : AF == OPURE_A_F16 ? 0x7E007E00u : 0x7FC07FC0u;
                const bool gone = (T::NB > 1u && r >= 8u ? pb : pa) < 0;
#pragma unroll
                for (uint32_t t = 0; t < T::NB; ++t)
#pragma unroll
                    for (uint32_t s = 0; s < T::KS; ++s) tl.k[t][s] = gone ? u4v{nan, nan, nan, nan} : tl.k[t][s];
            }
            // every row sees every position
            const bool full = t0 + TT <= min(sq.ctx + j0 + 1u, sq.total) && (t0 + TT <= p.sinks || t0 + p.window > sq.ctx + j1) && pa >= 0 && pb >= 0;
            float s[NT][NS];
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) win_scores<AF, HD>(p, tl, q[n], c, full, t0, g, sq.ctx + jr[n], sq.total, s[n]);
            if (more) tl.template load_k<ONCE>(at(na), at(nb), r, g);
            if (p.scores)
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n)
                    if (q0 + 16u * n + r < Gq)
                    {
                        float* to = p.scores + (((static_cast<uint64_t>(b) * p.n_kv + kh) * p.tiles + i) * Gq + q0 + 16u * n + r) * TT + NS * g;
#pragma unroll
                        for (uint32_t x = 0; x < NS; x += 4u) *reinterpret_cast<f4_t*>(to + x) = f4_t{s[n][x], s[n][x + 1], s[n][x + 2], s[n][x + 3]};
                    }
            u4v hi[NT], lo[NT];
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
            {
                float mx = s[n][0];
#pragma unroll
                for (uint32_t x = 1; x < NS; ++x) mx = fmaxf(mx, s[n][x]);
                mx = fmaxf(m[n], max_xor32(max_xor16(mx)));
                const float ms = mx == NEG_INF ? 0.0f : mx;
                const float a = __builtin_amdgcn_exp2f(__fsub_rn(m[n], ms));
                m[n] = mx;
                float sum = 0.0f;
#pragma unroll
                for (uint32_t x = 0; x < NS; ++x)
                {
                    s[n][x] = __builtin_amdgcn_exp2f(__fsub_rn(s[n][x], ms));
                    sum += s[n][x];
                }
                l[n] = __fmaf_rn(l[n], a, sum);                // this lane's share of the row's sum
#pragma unroll
                for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
                    for (uint32_t x = 0; x < 4; ++x) o[d][n][x] = __fmul_rn(o[d][n][x], a);
                if constexpr (AF == OPURE_A_F32)
                    hi[n] = u4v{f_bits(s[n][0]), f_bits(s[n][1]), f_bits(s[n][2]), f_bits(s[n][3])};
                else
#pragma unroll
                    for (uint32_t x = 0; x < 4; ++x)
                    {
                        hi[n][x] = win_pack<AF>(s[n][2 * x], s[n][2 * x + 1]);
                        lo[n][x] = win_pack<AF>(__fsub_rn(s[n][2 * x], win_low<AF>(hi[n][x])), __fsub_rn(s[n][2 * x + 1], win_high<AF>(hi[n][x])));
                    }
            }
            if (t0 + TT > sq.total || pa < 0 || pb < 0)
            {
                // slots past the sequence and pages that are not there hold anything: 0
                const uint32_t t = t0 + NS * g;
                const bool gone = (T::NB > 1u && g >= 2u ? pb : pa) < 0;
#pragma unroll
                for (uint32_t d = 0; d < DT; ++d) tl.v[d] = win_tail<AF>(tl.v[d], gone || t >= sq.total ? 0u : sq.total - t);
            }
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n)
                {
                    if constexpr (AF != OPURE_A_F32) o[d][n] = win_mfma<AF>(tl.v[d], lo[n], o[d][n]);
                    o[d][n] = win_mfma<AF>(tl.v[d], hi[n], o[d][n]);
                }
            if (!more) break;
            tl.template load_v<ONCE>(at(na) + vofs, at(nb) + vofs, r, g);
            pa = na;
            pb = nb;
            i += 4u;
        }
    }
    // ---- the waves' results through LDS, merged in wave order: wave w takes
    //      channel tiles w, w + 4, ... of every block
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
    {
        l[n] = add_xor32(add_xor16(l[n]));
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d) cacc[((wave * DT + d) * NT + n) * 64u + lane] = o[d][n];
        if (g == 0u)
        {
            cml[((wave * NT + n) * 16u + r) * 2u] = m[n];
            cml[((wave * NT + n) * 16u + r) * 2u + 1u] = l[n];
        }
    }
    __syncthreads();
    const uint64_t pbase = (((static_cast<uint64_t>(b) * p.n_kv + kh) * p.blocks + blk) * p.parts + part) * p.block_rows;
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
    {
        const uint32_t qi = 16u * n + r;                     // of the block
        float mw[4], w[4], M = NEG_INF, L = 0.0f;
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x)
        {
            mw[x] = cml[((x * NT + n) * 16u + r) * 2u];
            M = fmaxf(M, mw[x]);
        }
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x)
        {
            w[x] = __builtin_amdgcn_exp2f(__fsub_rn(mw[x], M == NEG_INF ? 0.0f : M));
            L = __fmaf_rn(w[x], cml[((x * NT + n) * 16u + r) * 2u + 1u], L);
        }
        if (q0 + qi >= Gq) continue;
        if (wave == 0u && g == 0u)
        {
            p.part_ml[(pbase + qi) * 2u] = M;
            p.part_ml[(pbase + qi) * 2u + 1u] = L;
        }
        for (uint32_t d = wave; d < DT; d += 4u)
        {
            f4_t acc = cacc[(d * NT + n) * 64u + lane];
#pragma unroll
            for (uint32_t i4 = 0; i4 < 4; ++i4) acc[i4] = __fmul_rn(w[0], acc[i4]);
#pragma unroll
            for (uint32_t x = 1; x < 4; ++x)
            {
                const f4_t v = cacc[((x * DT + d) * NT + n) * 64u + lane];
#pragma unroll
                for (uint32_t i4 = 0; i4 < 4; ++i4) acc[i4] = __fmaf_rn(w[x], v[i4], acc[i4]);
            }
            *reinterpret_cast<f4_t*>(p.part_acc + (pbase + qi) * HD + 16u * d + 4u * g) = acc;
        }
    }
}

// A query row's maximum M and sum L over its parts, lane x holding part x's.
__device__ __forceinline__ void win_total(float m, float l, uint32_t parts, uint32_t lane, float& M, float& w, float& L)
{
    M = wave_max64(lane < parts ? m : NEG_INF);
    w = lane < parts ? __builtin_amdgcn_exp2f(__fsub_rn(m, M == NEG_INF ? 0.0f : M)) : 0.0f;
    L = wave_sum64(lane < parts ? __fmul_rn(w, l) : 0.0f);
}

// Joins the parts: a workgroup a query row (WIDE: many parts, a wave every fourth
// one) or four rows (a wave each); DPL channels a lane.  A lane takes a part's
// maximum and sum, then channels.  Loads are unconditional (past the last part
// the last one again, weight 0): the code stays small, and a launch this short
// pays for every line of it (3.5 us for one row of 32 heads in 9 parts, 7.2 with
// each load under its test).  A row that is not finite is computed again position
// by position: a NaN or an infinity among the values of a position that the row
// does not see meets weight 0 in the products above.  With scores, the launch's
// other workgroups add the weights: PPT positions a thread (one where there are
// few), over the query rows in order, 32 / PPT rows' maxima and sums at a time.
//   A launch of its own: joining in the workgroup that arrives last needs fences
// across the XCDs, which cost more than the launch (one row over 1,000 positions
// 7.9 us in two launches, 9.5 in one; the 32 sequences above 78 and 433).
template <uint32_t TT, bool WIDE, uint32_t DPL, uint32_t PPT>
__global__ __launch_bounds__(256) void k_win_join(WinParams p)
{
    __shared__ float sm[4][256];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, G = p.n_heads / p.n_kv, Gq = G * p.rows;
    const uint32_t shift = p.two ? 5u : 4u;                // a block's query rows
    if (blockIdx.x < p.combine_wgs)
    {
        const uint32_t id = WIDE ? blockIdx.x : 4u * blockIdx.x + wave;
        if (id >= p.combine_rows) return;                  // never with WIDE: the barrier below
        const uint32_t row = id / p.n_heads, head = id - row * p.n_heads, b = row / p.rows, j = row - b * p.rows;
        const uint32_t kh = head / G, qi = j * G + (head - kh * G), blk = qi >> shift, qb = qi - (blk << shift);
        const uint32_t parts = p.parts, end = parts - 1u;
        const uint64_t slot = ((static_cast<uint64_t>(b) * p.n_kv + kh) * p.blocks + blk) * parts;
        const uint64_t ml = ((slot + min(lane, end)) * p.block_rows + qb) * 2u;
        const float pm = p.part_ml[ml], pl = p.part_ml[ml + 1u];
        constexpr uint32_t U = WIDE ? 8u : 4u, BY = WIDE ? 4u : 1u;
        const uint32_t x0 = WIDE ? wave : 0u;
        float v[U][DPL], o[DPL];
        auto fetch = [&](uint32_t x) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t i = 0; i < DPL; ++i)
                    v[u][i] = p.part_acc[((slot + min(x + BY * u, end)) * p.block_rows + qb) * p.hd + min(lane + 64u * i, p.hd - 1u)];
        };
        fetch(x0);
        float M, w, L;
        win_total(pm, pl, parts, lane, M, w, L);
#pragma unroll
        for (uint32_t i = 0; i < DPL; ++i) o[i] = 0.0f;
        for (uint32_t x = x0; x < parts; x += BY * U)
        {
            if (x != x0) fetch(x);
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
            {
                const uint32_t y = x + BY * u;
                const float wx = y < parts ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), min(y, 63u))) : 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < DPL; ++i) o[i] = __fmaf_rn(wx, v[u][i], o[i]);
            }
        }
        if constexpr (WIDE)
        {
#pragma unroll
            for (uint32_t i = 0; i < DPL; ++i) sm[wave][lane + 64u * i] = o[i];
            __syncthreads();
            if (wave != 0u) return;
#pragma unroll
            for (uint32_t i = 0; i < DPL; ++i) o[i] = (sm[0][lane + 64u * i] + sm[1][lane + 64u * i]) + (sm[2][lane + 64u * i] + sm[3][lane + 64u * i]);
            __builtin_amdgcn_wave_barrier();
        }
        if (p.lse && lane == 0u) p.lse[(static_cast<uint64_t>(b) * p.n_kv + kh) * Gq + qi] = win_lse(M, L);
        bool fine = true;
#pragma unroll
        for (uint32_t i = 0; i < DPL; ++i)
        {
            o[i] = L == 0.0f ? 0.0f : __fdiv_rn(o[i], L);
            fine = fine && (__builtin_isfinite(o[i]) || lane + 64u * i >= p.hd);
        }
        const uint64_t at = static_cast<uint64_t>(id) * p.hd;
        if (!__all(fine))
        {
            for (uint32_t d = lane; d < p.hd; d += 64u) sm[wave][d] = load_act_rt(p.q, at + d, p.afmt);
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const WinSeq sq = win_seq(p, p.seq_len[b]);
            float m, l, x[4];
            win_row(p, sm[wave], b, kh, sq.ctx + j, sq.total, m, l, x);
#pragma unroll
            for (uint32_t i = 0; i < DPL; ++i) o[i] = l == 0.0f ? 0.0f : __fdiv_rn(x[i], l);
        }
#pragma unroll
        for (uint32_t i = 0; i < DPL; ++i)
            if (lane + 64u * i < p.hd) store_act_rt(p.out, at + lane + 64u * i, o[i], p.afmt);
        return;
    }
    // ---- weights: 256 PPT positions of a (sequence, KV head)
    typedef float vec_t __attribute__((ext_vector_type(PPT)));
    const uint32_t per = (p.tiles * TT + 256u * PPT - 1u) / (256u * PPT), id = blockIdx.x - p.combine_wgs;
    const uint32_t bh = id / per, x = id - bh * per, b = bh / p.n_kv, kh = bh - b * p.n_kv;
    const WinSeq sq = win_seq(p, p.seq_len[b]);
    const WinSpan span = win_span<TT>(p, sq, sq.ctx, sq.ctx + p.rows);
    if (x * 256u * PPT >= span.n * TT) return;                // whole workgroup
    const uint32_t at = (x * 256u + threadIdx.x) * PPT, i = min(at / TT, span.n - 1u), off = at % TT;
    const uint32_t t = at < span.n * TT ? span.tile(i) * TT + off : sq.total;
    const float* s = p.scores + (static_cast<uint64_t>(bh) * p.tiles + i) * Gq * TT + off;
    float* to = p.weights + b * p.weights_batch_stride + static_cast<uint64_t>(kh) * p.weights_stride + t;
    float sum[PPT], old[PPT];
    bool any[PPT];
#pragma unroll
    for (uint32_t k = 0; k < PPT; ++k)
    {
        sum[k] = 0.0f;
        any[k] = false;
        old[k] = t + k < sq.total ? to[k] : 0.0f;
    }
    uint32_t j = 0, g = 0;                                    // the query row's row and head
    constexpr uint32_t U = 8u / PPT, C = 4u * U;              // rows a wave; a turn
    for (uint32_t c0 = 0; c0 < Gq; c0 += C)
    {
        vec_t v[C];
        float pm[U], pl[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            if (c0 + 4u * u < Gq)
            {
                const uint32_t qi = min(c0 + 4u * u + wave, Gq - 1u), blk = qi >> shift;
                const uint64_t slot = (static_cast<uint64_t>(bh) * p.blocks + blk) * p.parts + min(lane, p.parts - 1u);
                const uint64_t ml = (slot * p.block_rows + (qi - (blk << shift))) * 2u;
                pm[u] = p.part_ml[ml];
                pl[u] = p.part_ml[ml + 1u];
            }
#pragma unroll
        for (uint32_t y = 0; y < C; ++y)
            if (c0 + y < Gq) v[y] = *reinterpret_cast<const vec_t*>(s + static_cast<uint64_t>(c0 + y) * TT);
        if (c0) __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            if (c0 + 4u * u < Gq)
            {
                float M, w, L;
                win_total(pm[u], pl[u], p.parts, lane, M, w, L);
                if (lane == 0u)
                {
                    sm[0][4u * u + wave] = M == NEG_INF ? 0.0f : M;
                    sm[1][4u * u + wave] = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
                }
            }
        __syncthreads();
#pragma unroll
        for (uint32_t y = 0; y < C; ++y)
            if (c0 + y < Gq)
            {
                const float m = sm[0][y], inv = sm[1][y];
#pragma unroll
                for (uint32_t k = 0; k < PPT; ++k)
                {
                    const bool sees = t + k < sq.total && win_sees(p, sq.ctx + j, t + k);
                    any[k] = any[k] || sees;
                    sum[k] += sees ? __fmul_rn(__builtin_amdgcn_exp2f(__fsub_rn(v[y][k], m)), inv) : 0.0f;
                }
                const bool wrap = g + 1u == G;
                g = wrap ? 0u : g + 1u;
                j += wrap ? 1u : 0u;
            }
    }
#pragma unroll
    for (uint32_t k = 0; k < PPT; ++k)
        if (any[k]) to[k] = old[k] + sum[k];
}

template <int HD, int NT>
constexpr uint32_t win_split_lds() { return 4u * (HD / 16u) * NT * 64u * 16u + 4u * NT * 16u * 2u * 4u; }

// f(kernel, dynamic LDS, workgroups of it that the device holds at a time) for a head size and format.
// What a CU holds is asked once a kernel: it is the same on every device that the code is built for.
template <typename F>
int win_split_kernel(opure_dev* dev, uint32_t afmt, uint32_t hd, bool two, bool once, F&& f)
{
    auto one = [&](auto af, auto h, auto nt, auto alone) {
        constexpr int AF = decltype(af)::value, HD = decltype(h)::value, NT = decltype(nt)::value;
        constexpr bool ONCE = decltype(alone)::value;
        static std::atomic<uint64_t> done{0};
        static std::atomic<int> a_cu{0};
        auto* kernel = &k_win_split<AF, HD, NT, ONCE>;
        const int rc = win_lds(dev, reinterpret_cast<const void*>(kernel), win_split_lds<HD, NT>(), done);
        if (rc) return rc;
        int n = a_cu.load(std::memory_order_relaxed);
        if (n == 0)
        {
            OPURE_HIP_TRY(hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, win_split_lds<HD, NT>()));
            n = std::max(n, 1);
            a_cu.store(n, std::memory_order_relaxed);
        }
        return f(kernel, win_split_lds<HD, NT>(), static_cast<uint32_t>(n) * (dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u));
    };
    auto by_head = [&](auto af) {
        return win_by_head(hd, [&](auto h) {
            if constexpr (decltype(h)::value <= 128)
            {
                if (two) return one(af, h, std::integral_constant<int, 2>{}, std::false_type{});
            }
            else if (!once) return one(af, h, std::integral_constant<int, 1>{}, std::false_type{});
            return one(af, h, std::integral_constant<int, 1>{}, std::true_type{});
        });
    };
    return afmt == OPURE_A_F32   ? by_head(std::integral_constant<int, OPURE_A_F32>{})
           : afmt == OPURE_A_F16 ? by_head(std::integral_constant<int, OPURE_A_F16>{})
                                 : by_head(std::integral_constant<int, OPURE_A_BF16>{});
}

// How a call is split, and its workspace.
struct WinPlan {
    uint32_t tt = 0, tiles = 0, blocks = 0, block_rows = 0, parts = 0;
    bool prompt = false;                                 // the prompt kernel
    bool two = false, stored = false, four = false;      // split: 32 query rows a workgroup; weights from stored scores, four positions a thread
    uint64_t acc = 0, ml = 0, scores = 0, lse = 0, sums = 0;   // bytes
    uint64_t bytes() const { return acc + ml + scores + lse + sums; }
};

// Which kernels take a call, by what each would take (us, of what was measured on
// 8 KV heads of 64, 128 and 192 channels and 4 of 256, 2 or 4 query heads each):
//   k_win_prompt walks all tiles of 64 positions in one workgroup a 128 query rows:
//     3 + channels / 32, and a tile 0.4 + channels / 125 (past 128 channels, without
//     two waves a row block, channels / 60), times the workgroups a CU;
//   k_win_split + k_win_join: 7 + channels / 100, 1.1 ns a tile of 32 positions, block
//     of query rows and 100 channels, and 0.3 a query row and 100,000 channels of it.
// Measured, prompt / split: 64 query rows of a KV head over 64 positions 5.8 / 7.6 (of
// 128 channels 8.4 / 8.5, of 256 12.0 / 9.3), over 1,000 19.1 / 8.3, over 8,000 115.6 /
// 13.1; four sequences of 512 over 1,000 21.4 / 16.5, of 1,024 24.9 / 50.3; 1,024 of
// 128 channels behind a window of 1,024 33.4 / 25.5, over 1,000 in four sequences
// 40.3 / 74.8.  Of 184 such calls it takes the slower one in 6, by 1.5 us at most.
//   Weights from stored scores cost the join 0.2 a query row, or its scores' 8 bytes a
// position, written and read, at 5.3 TB/s; computed again (k_win_sums) they cost 2 +
// channels / 64 and the keys once more at 2.5 TB/s.  Measured, stored / computed again:
// 16 query rows over 500 positions of 64 channels 9.9 / 11.4, 64 20.4 / 13.0, 64 over
// 4,000 in 16 sequences 104 / 87; of 128 channels 22.2 / 16.0, 141 / 177, of 256 22.0 /
// 19.9, 229 / 250.  Stored scores are workspace too: past 64 MB no more than the keys
// that they save reading, and no more rows than the 96 that were measured.
void win_choose(const opure_dev* dev, const opure_attn_window_args* a, WinPlan& w)
{
    const opure_model* m = a->model;
    const double G = m->n_heads / m->n_kv_heads, Gq = G * a->rows, hd = m->head_dim, cu = dev->n_cu > 0 ? dev->n_cu : 256;
    const double heads = static_cast<double>(a->batch) * m->n_kv_heads, span = static_cast<double>(w.tiles) * w.tt;
    const double wgs = heads * std::ceil(Gq / 128.0), window = a->window ? a->window : 2147483647.0;
    const double prompt = 3.0 + hd / 32.0 + std::max(1.0, wgs / cu) * std::ceil(std::min(span, a->sinks + window + 128.0 / G) / 64.0) *
                                                (hd <= 128.0 ? 0.4 + hd / 125.0 : hd / 60.0);
    const double split = 7.0 + hd / 100.0 + heads * hd * (std::ceil(Gq / (Gq > 16.0 && hd <= 128.0 ? 32.0 : 16.0)) * w.tiles * 1.1e-5 + Gq * 3e-6);
    const double keys = heads * span * hd * act_bytes(m->afmt), scores = heads * span * 4.0 * Gq;
    const double store = std::max(0.2 * Gq, 2.0 * scores / 5.3e6), again = 2.0 + hd / 64.0 + keys / 2.5e6;
    w.stored = a->weights && Gq <= 96.0 && store < again && scores <= std::max(67108864.0, keys);
    w.prompt = m->afmt != OPURE_A_F32 && prompt + (a->weights ? again : 0.0) < split + (w.stored ? store : a->weights ? again : 0.0);
    if (w.prompt) w.stored = false;
}

int win_plan(opure_dev* dev, const opure_attn_window_args* a, WinPlan& w)
{
    const opure_model* m = a->model;
    const uint32_t Gq = m->n_heads / m->n_kv_heads * a->rows;
    w.tt = m->afmt == OPURE_A_F32 ? 16u : 32u;
    // tiles of any sequence of the call: its sinks', then the window's and the rows', which begin anywhere in a tile
    const uint64_t all = (a->max_ctx + w.tt - 1u) / w.tt, window = a->window ? a->window : 0x7FFFFFFFu;
    w.tiles = static_cast<uint32_t>(std::min<uint64_t>(all, (a->sinks + w.tt - 1ull) / w.tt + (window + a->rows + w.tt - 2ull) / w.tt + 1u));
    const uint64_t rows = static_cast<uint64_t>(a->batch) * m->n_kv_heads * Gq;
    win_choose(dev, a, w);
    w.lse = a->weights && !w.stored ? opure_hip::align_up(rows * 4u, 256) : 0u;
    uint64_t most = 0;                                   // workgroups of the call's largest launch
    if (w.lse)
    {
        WinParams p{};
        p.n_heads = m->n_heads;
        p.n_kv = m->n_kv_heads;
        p.rows = a->rows;
        p.cap = a->max_ctx;
        p.afmt = m->afmt;
        w.sums = win_sums_bytes(dev, p, a->batch);
        most = win_sums_workgroups(dev, p, a->batch);
    }
    // a launch's threads, 256 a workgroup, stay in 32 bits
    auto fits = [&](uint64_t wgs) {
        OPURE_REQUIRE(std::max(wgs, most) < 1u << 24, OPURE_E_CAPACITY,
                      "window attention: %u x %u rows of %u heads over max_ctx %u: too many workgroups", a->batch, a->rows, m->n_heads, a->max_ctx);
        return OPURE_OK;
    };
    const uint64_t heads = static_cast<uint64_t>(a->batch) * m->n_kv_heads;
    if (w.prompt) return fits(heads * ((Gq + 127u) / 128u));
    w.two = Gq > 16u && m->head_dim <= 128u;
    w.blocks = (Gq + (w.two ? 31u : 15u)) / (w.two ? 32u : 16u);
    w.block_rows = std::min(Gq, w.two ? 32u : 16u);
    uint32_t room = 0;
    const int rc = win_split_kernel(dev, m->afmt, m->head_dim, w.two, w.blocks == 1u, [&](auto, uint32_t, uint32_t n) {
        room = n;
        return OPURE_OK;
    });
    if (rc) return rc;
    const uint64_t groups = heads * w.blocks;
    // Parts of a group: as many as the device holds at a time, each of at least four tiles (one a wave), or of so many
    // that the part's outputs, written and read again, stay a quarter of its keys and values (24 rows of 8B heads over
    // 66 tiles: 16 parts 26.9 us, 11 24.9, 8 24.7); three times as many where a wave still has four tiles, which evens
    // out ragged sequences (16 sequences of 2,000 to 8,000: 2 parts 91.5 us, 4 77.6, 12 73.4)
    const uint32_t least = std::max(4u, w.block_rows / 4u);
    const uint64_t fill = std::max<uint64_t>(1u, room / groups), more = std::min<uint64_t>(3ull * room / groups, w.tiles / 16u);
    w.parts = static_cast<uint32_t>(std::min<uint64_t>(std::max(fill, more), std::min((w.tiles + least - 1u) / least, MAX_PARTS)));
    const uint64_t wide = heads * ((static_cast<uint64_t>(w.tiles) * w.tt + 1023u) / 1024u);
    w.four = wide >= 2ull * (dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u);
    const uint64_t slots = groups * w.parts * w.block_rows;
    w.acc = opure_hip::align_up(slots * m->head_dim * 4u, 256);
    w.ml = opure_hip::align_up(slots * 8u, 256);
    w.scores = w.stored ? opure_hip::align_up(rows * w.tiles * w.tt * 4u, 256) : 0u;
    // the join's: a row a workgroup or four, and with stored scores 1,024 positions or 256
    const uint64_t join = (w.parts > 8u ? rows : (rows + 3u) / 4u) + (w.stored ? (w.four ? wide : 4u * wide) : 0u);
    return fits(std::max(groups * w.parts, join));
}

int win_validate(const opure_attn_window_args* a)
{
    OPURE_REQUIRE(a && a->model && a->kv && a->kv->pool && a->kv->page_table, OPURE_E_INVALID,
                  "window attention: null argument, model or cache");
    const opure_model* m = a->model;
    const opure_kv* kv = a->kv;
    OPURE_REQUIRE(m->n_kv_heads >= 1 && m->n_heads >= 1 && m->n_heads % m->n_kv_heads == 0, OPURE_E_INVALID,
                  "window attention: n_heads %u %% n_kv_heads %u != 0", m->n_heads, m->n_kv_heads);
    OPURE_REQUIRE(m->head_dim >= 16 && m->head_dim <= 256 && m->head_dim % 16 == 0, OPURE_E_UNSUPPORTED,
                  "window attention: head_dim %u not in 16..256 step 16", m->head_dim);
    OPURE_REQUIRE(m->afmt <= OPURE_A_BF16, OPURE_E_INVALID, "window attention: bad activation format");
    OPURE_REQUIRE(kv->page_size == OPURE_PAGE_SIZE, OPURE_E_UNSUPPORTED, "window attention: page_size must be %d",
                  OPURE_PAGE_SIZE);
    OPURE_REQUIRE(kv->n_pages >= 1 && kv->max_pages_per_seq >= 1, OPURE_E_INVALID, "window attention: the cache has no pages");
    OPURE_REQUIRE(a->layer < m->n_layers, OPURE_E_INVALID, "window attention: layer %u of %u", a->layer, m->n_layers);
    OPURE_REQUIRE(a->batch >= 1 && a->batch <= OPURE_MAX_BATCH_ROWS && a->rows >= 1 && a->rows <= OPURE_MAX_PROMPT_ROWS,
                  OPURE_E_CAPACITY, "window attention: %u rows x %u sequences outside 1..%d x 1..%d", a->rows, a->batch,
                  OPURE_MAX_PROMPT_ROWS, OPURE_MAX_BATCH_ROWS);
    // the query rows' indexes stay in 32 bits
    OPURE_REQUIRE(static_cast<uint64_t>(m->n_heads) * a->batch * a->rows <= 1u << 25, OPURE_E_CAPACITY,
                  "window attention: %u x %u rows of %u heads", a->batch, a->rows, m->n_heads);
    const uint64_t slots = static_cast<uint64_t>(kv->max_pages_per_seq) * OPURE_PAGE_SIZE;
    OPURE_REQUIRE(a->max_ctx >= a->rows && a->max_ctx <= slots && a->max_ctx <= 0x7FFFFFFFu - OPURE_MAX_PROMPT_ROWS,
                  OPURE_E_CAPACITY, "window attention: max_ctx %u below %u rows or beyond the page table's %llu", a->max_ctx,
                  a->rows, (unsigned long long)slots);
    OPURE_REQUIRE(a->sinks <= 0x7FFFFFFFu, OPURE_E_INVALID, "window attention: %u sinks", a->sinks);
    OPURE_REQUIRE(!a->weights || a->weights_stride >= a->max_ctx, OPURE_E_INVALID,
                  "window attention: weights_stride %u below max_ctx %u", a->weights_stride, a->max_ctx);
    OPURE_REQUIRE(!a->weights || a->batch == 1u ||
                      a->weights_batch_stride >= static_cast<uint64_t>(m->n_kv_heads - 1u) * a->weights_stride + a->max_ctx,
                  OPURE_E_INVALID, "window attention: weights_batch_stride %llu: sequences overlap",
                  (unsigned long long)a->weights_batch_stride);
    OPURE_REQUIRE((reinterpret_cast<uintptr_t>(kv->pool) & 15u) == 0u && (reinterpret_cast<uintptr_t>(kv->page_table) & 3u) == 0u,
                  OPURE_E_INVALID, "window attention: pool must be 16-byte aligned, page_table 4-byte");
    return OPURE_OK;
}

}  // namespace

using namespace opure_hip;

extern "C" int opure_attn_window_reserve(opure_dev* dev, const opure_attn_window_args* a)
{
    OPURE_REQUIRE(dev, OPURE_E_INVALID, "opure_attn_window_reserve: null device");
    const int rc = win_validate(a);
    if (rc) return rc;
    const DeviceGuard on(dev);
    WinPlan w;
    const int rp = win_plan(dev, a, w);
    return rp ? rp : ensure_workspace(dev, w.bytes());
}

extern "C" int opure_attn_window_paged(opure_dev* dev, const opure_attn_window_args* a)
{
    OPURE_REQUIRE(dev && a && a->q && a->out && a->seq_len, OPURE_E_INVALID, "opure_attn_window_paged: null argument");
    int rc = win_validate(a);
    if (rc) return rc;
    OPURE_REQUIRE((reinterpret_cast<uintptr_t>(a->q) & 15u) == 0u && (reinterpret_cast<uintptr_t>(a->out) & 7u) == 0u &&
                      ((reinterpret_cast<uintptr_t>(a->seq_len) | reinterpret_cast<uintptr_t>(a->weights)) & 3u) == 0u,
                  OPURE_E_INVALID, "opure_attn_window_paged: q must be 16-byte aligned, out 8-byte, seq_len and weights 4-byte");
    const opure_model* m = a->model;
    const uint64_t bytes = static_cast<uint64_t>(a->batch) * a->rows * m->n_heads * m->head_dim * act_bytes(m->afmt);
    const uint64_t cache = static_cast<uint64_t>(m->n_layers) * a->kv->n_pages * 2u * m->n_kv_heads * OPURE_PAGE_SIZE * m->head_dim * act_bytes(m->afmt);
    const uint64_t table = static_cast<uint64_t>(a->batch) * a->kv->max_pages_per_seq * 4u;
    const uint64_t spread = ((a->batch - 1u) * a->weights_batch_stride + static_cast<uint64_t>(m->n_kv_heads - 1u) * a->weights_stride + a->max_ctx) * 4u;
    OPURE_REQUIRE(!overlaps(a->out, bytes, a->q, bytes), OPURE_E_INVALID, "opure_attn_window_paged: out overlaps q");
    OPURE_REQUIRE(!overlaps(a->out, bytes, a->kv->pool, cache) && !overlaps(a->out, bytes, a->kv->page_table, table) &&
                      !overlaps(a->out, bytes, a->seq_len, a->batch * 4u), OPURE_E_INVALID, "opure_attn_window_paged: out overlaps the cache");
    OPURE_REQUIRE(!overlaps(a->weights, spread, a->q, bytes) && !overlaps(a->weights, spread, a->out, bytes) &&
                      !overlaps(a->weights, spread, a->kv->pool, cache) && !overlaps(a->weights, spread, a->kv->page_table, table) &&
                      !overlaps(a->weights, spread, a->seq_len, a->batch * 4u),
                  OPURE_E_INVALID, "opure_attn_window_paged: weights overlaps q, out or the cache");
    // the call's parts and scores go to the workspace, which may also move
    OPURE_REQUIRE(!overlaps(dev->ws, dev->ws_bytes, a->q, bytes) && !overlaps(dev->ws, dev->ws_bytes, a->out, bytes) &&
                      !overlaps(dev->ws, dev->ws_bytes, a->weights, spread),
                  OPURE_E_INVALID, "opure_attn_window_paged: q, out or weights in the device's workspace");
    const DeviceGuard on(dev);
    WinPlan w;
    rc = win_plan(dev, a, w);
    if (rc) return rc;
    rc = ensure_workspace(dev, w.bytes());
    if (rc) return rc;
    WinParams p{};
    p.q = a->q;
    p.out = a->out;
    p.pool = a->kv->pool;
    p.page_table = a->kv->page_table;
    p.seq_len = a->seq_len;
    p.part_acc = static_cast<float*>(dev->ws);
    p.part_ml = p.part_acc + w.acc / 4u;
    p.scores = w.stored ? p.part_ml + w.ml / 4u : nullptr;
    p.lse = w.lse ? p.part_ml + (w.ml + w.scores) / 4u : nullptr;
    float* const sums_at = w.lse ? p.lse + w.lse / 4u : nullptr;
    p.weights = a->weights;
    p.weights_stride = a->weights_stride;
    p.weights_batch_stride = a->weights_batch_stride;
    p.n_heads = a->model->n_heads;
    p.n_kv = a->model->n_kv_heads;
    p.hd = a->model->head_dim;
    p.rows = a->rows;
    p.n_pages = a->kv->n_pages;
    p.max_pages = a->kv->max_pages_per_seq;
    p.layer = a->layer;
    p.afmt = a->model->afmt;
    p.window = a->window == 0u || a->window > 0x7FFFFFFFu ? 0x7FFFFFFFu : a->window;
    p.sinks = a->sinks;
    p.cap = a->max_ctx;
    p.scale = a->model->attn_scale;
    p.err = dev->err;
    p.parts = w.parts;
    p.blocks = w.blocks;
    p.block_rows = w.block_rows;
    p.two = w.two ? 1u : 0u;
    p.tiles = w.tiles;
    p.combine_rows = a->batch * a->rows * p.n_heads;
    if (w.prompt)
    {
        rc = win_prompt_launch(dev, p, a->batch);
        return rc || !p.lse ? rc : win_sums_launch(dev, p, a->batch, sums_at);
    }
    const uint32_t wgs = p.n_kv * w.parts * w.blocks * a->batch;
    rc = win_split_kernel(dev, p.afmt, p.hd, w.two, w.blocks == 1u, [&](auto kernel, uint32_t lds, uint32_t) {
        OPURE_LAUNCH(dev, kernel, dim3(wgs), dim3(256), lds, p);
        OPURE_LAUNCH_CHECK("k_win_split");
        return OPURE_OK;
    });
    if (rc) return rc;
    const uint32_t sums = p.scores ? (w.tiles * w.tt + (w.four ? 1023u : 255u)) / (w.four ? 1024u : 256u) * p.n_kv * a->batch : 0u;
    const bool wide = w.parts > 8u;
    p.combine_wgs = wide ? p.combine_rows : (p.combine_rows + 3u) / 4u;
    auto join = [&](auto tt, auto all, auto ppt) {
        constexpr uint32_t TT = decltype(tt)::value, PPT = decltype(ppt)::value;
        constexpr bool WIDE = decltype(all)::value;
        const dim3 grid(p.combine_wgs + sums), block(256);
        switch ((p.hd + 63u) / 64u)
        {
        case 1: OPURE_LAUNCH(dev, (k_win_join<TT, WIDE, 1, PPT>), grid, block, 0, p); break;
        case 2: OPURE_LAUNCH(dev, (k_win_join<TT, WIDE, 2, PPT>), grid, block, 0, p); break;
        case 3: OPURE_LAUNCH(dev, (k_win_join<TT, WIDE, 3, PPT>), grid, block, 0, p); break;
        default: OPURE_LAUNCH(dev, (k_win_join<TT, WIDE, 4, PPT>), grid, block, 0, p); break;
        }
    };
    typedef std::integral_constant<uint32_t, 1> One;
    typedef std::integral_constant<uint32_t, 4> Four;
    auto join_tt = [&](auto tt) {
        if (w.four) wide ? join(tt, std::true_type{}, Four{}) : join(tt, std::false_type{}, Four{});
        else wide ? join(tt, std::true_type{}, One{}) : join(tt, std::false_type{}, One{});
    };
    if (w.tt == 16u) join_tt(std::integral_constant<uint32_t, 16>{});
    else join_tt(std::integral_constant<uint32_t, 32>{});
    OPURE_LAUNCH_CHECK("k_win_join");
    return p.lse ? win_sums_launch(dev, p, a->batch, sums_at) : OPURE_OK;
}
