// ============================================================================
//  kv4_attn.hip -- attention over the 4-bit paged cache (kv4.h), with a sliding
//  window and first positions that stay visible or without.
//
//  Row j of a sequence, at position p = seq_len + j, sees t <= p with t < sinks or
//  t > p - window:  s_t = scale q.k_t,  w_t = exp(s_t - m) / sum exp(s - m),
//  out = sum w_t v_t.
// ============================================================================
#include "kv4_attn.h"

using namespace opure_kv4;
using opure_hip::act_bytes;

namespace {

// A workgroup takes a piece of the tiles that the sequences' rows see, for 16 NT query
// rows of a KV head, a wave every fourth tile.  The four waves are merged in LDS, the
// parts by k_kv4_join.
//   PIECES: of one size over all sequences, where they are long; else a workgroup has a
// part of one sequence, as many of each.
//   Bound by memory and, close behind, the vector unit (3 instructions a pair of codes, the
// softmax; 63% of the clocks): 32 sequences of 1,024 to 16,384 positions, 8 KV heads of 128,
// 232 MB in 53 us with the join, 4.4 TB/s (49 us this kernel, 4.7 TB/s, a large copy's rate).
// A single sequence of 2,000 is launches and round trips, 4.4 and 3.3 us.  Three waves a SIMD
// at up to 128 channels, which have 168 registers each (a form that spilled some took 66 us for
// 57), one past that; of fp32 rows, which are two numbers each, two (that batch 57 us).
template <int AF, int HD, int NT, bool ONCE, bool PIECES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NT == 2 ? 2 : HD > 128 ? 1 : AF == OPURE_A_F32 ? 2 : 3))) void k_kv4_split(WinParams p)
{
    constexpr uint32_t DT = HD / 16u;
    extern __shared__ __align__(16) uint8_t lds[];
    f4_t* cacc = reinterpret_cast<f4_t*>(lds);                            // [wave][DT][NT][64]
    float* cml = reinterpret_cast<float*>(lds + 4u * DT * NT * 64u * 16u);   // [wave][NT][16][2]
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // KV heads next to each other, then pieces, or parts, blocks of rows and sequences
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, part = PIECES ? rest : rest % p.parts, group = PIECES ? 0u : rest / p.parts;
    uint32_t b = ONCE ? group : group / p.blocks;
    const uint32_t blk = ONCE ? 0u : group - b * p.blocks;
    uint32_t before = 0, at0 = 0, at1 = 0;                 // tiles at0 .. at1 - 1 of all, those before sequence b
    if constexpr (PIECES)
    {
        const Share share = share_out<true>(p, part);
        at0 = part * share.size;
        if (at0 >= share.total) return;                    // pieces that the lengths leave over
        at1 = min(at0 + share.size, share.total);
        b = share.b;
        before = share.before;
    }
    Kv4Wave<AF, HD, NT, ONCE, 4u> w(p, kh, blk * 16u * NT);
    uint32_t has;
    auto start = [&]() {
        w.seek(b);
        has = max(w.span.n, 1u);
        if constexpr (PIECES) w.start(b, at0 - before + wave, min(min(at1 - before, has), w.span.n));
        else w.start(b, part_of(p, w.span.n * part) + wave, part_of(p, w.span.n * (part + 1u)));
    };
    start();
    while (true)
    {
        w.run();
        w.leave(wave, cacc, cml);
        const uint64_t slot = PIECES ? static_cast<uint64_t>(part + b) * p.n_kv + kh : ((static_cast<uint64_t>(b) * p.n_kv + kh) * p.blocks + blk) * p.parts + part;
        const uint64_t pbase = slot * p.block_rows;
        bool on = false;
        if constexpr (PIECES)
        {
            // the next sequence's loads on their way while this one's results are merged
            before += has;
            at0 = before;
            on = at0 < at1;
            if (on)
            {
                ++b;
                start();
            }
        }
        // merged in wave order: wave w takes channel tiles w, w + 4, ... of every block
        __syncthreads();
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
        {
            const uint32_t qi = 16u * n + w.r;                     // of the block
            float mw[4], f[4], M = NEG_INF, L = 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
            {
                mw[x] = cml[((x * NT + n) * 16u + w.r) * 2u];
                M = fmaxf(M, mw[x]);
            }
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
            {
                f[x] = __builtin_amdgcn_exp2f(__fsub_rn(mw[x], M == NEG_INF ? 0.0f : M));
                L = __fmaf_rn(f[x], cml[((x * NT + n) * 16u + w.r) * 2u + 1u], L);
            }
            if (w.q0 + qi >= w.Gq) continue;
            if (wave == 0u && w.g == 0u)
            {
                p.part_ml[(pbase + qi) * 2u] = M;
                p.part_ml[(pbase + qi) * 2u + 1u] = L;
            }
            for (uint32_t d = wave; d < DT; d += 4u)
            {
                f4_t acc = cacc[(d * NT + n) * 64u + w.lane];
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y) acc[y] = __fmul_rn(f[0], acc[y]);
#pragma unroll
                for (uint32_t x = 1; x < 4; ++x)
                {
                    const f4_t v = cacc[((x * DT + d) * NT + n) * 64u + w.lane];
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) acc[y] = __fmaf_rn(f[x], v[y], acc[y]);
                }
                *reinterpret_cast<f4_t*>(p.part_acc + (pbase + qi) * HD + 16u * d + 4u * w.g) = acc;
            }
        }
        if (!on) return;
        __syncthreads();                                       // the merge has read the waves' results
    }
}

// Joins the parts: a workgroup a query row (WIDE: many parts, a wave every fourth
// one) or four rows (a wave each); DPL channels a lane.  A row that is not finite is
// computed again position by position: a NaN among the values of a position that the
// row does not see meets weight 0 in the products above.
template <bool WIDE, uint32_t DPL>
__global__ __launch_bounds__(256) void k_kv4_join(WinParams p)
{
    __shared__ float sm[4][256];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, G = p.n_heads / p.n_kv;
    const uint32_t shift = p.two == 2u ? 7u : p.two ? 5u : 4u;   // a block's query rows
    const uint32_t id = WIDE ? blockIdx.x : 4u * blockIdx.x + wave;
    if (id >= p.combine_rows) return;                      // never with WIDE: the barrier below
    const uint32_t row = id / p.n_heads, head = id - row * p.n_heads, b = row / p.rows, j = row - b * p.rows;
    const uint32_t kh = head / G, qi = j * G + (head - kh * G), blk = qi >> shift, qb = qi - (blk << shift);
    // part x's slot is slot + x * step
    uint32_t parts = p.parts;
    uint64_t step = 1u, slot = ((static_cast<uint64_t>(b) * p.n_kv + kh) * p.blocks + blk) * parts;
    if (p.pieces)
    {
        // the pieces that hold the sequence's first and last tile
        const Share share = share_out<false>(p, b);
        const uint32_t piece = share.before / share.size;
        parts = (share.before + seq_tiles(p, b) - 1u) / share.size - piece + 1u;
        step = p.n_kv;
        slot = (piece + b) * step + kh;
    }
    const uint32_t end = parts - 1u;
    const uint64_t ml = ((slot + min(lane, end) * step) * p.block_rows + qb) * 2u;
    const float pm = p.part_ml[ml], pl = p.part_ml[ml + 1u];
    constexpr uint32_t U = WIDE ? 8u : 4u, BY = WIDE ? 4u : 1u;
    const uint32_t x0 = WIDE ? wave : 0u;
    float v[U][DPL], o[DPL];
    auto fetch = [&](uint32_t x) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
#pragma unroll
            for (uint32_t i = 0; i < DPL; ++i)
                v[u][i] = p.part_acc[((slot + min(x + BY * u, end) * step) * p.block_rows + qb) * p.hd + min(lane + 64u * i, p.hd - 1u)];
    };
    fetch(x0);
    const float M = wave_max64(lane < parts ? pm : NEG_INF);
    const float w = lane < parts ? __builtin_amdgcn_exp2f(__fsub_rn(pm, M == NEG_INF ? 0.0f : M)) : 0.0f;
    const float L = wave_sum64(lane < parts ? __fmul_rn(w, pl) : 0.0f);
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
        float l, x[4];
        kv4_row(p, sm[wave], b, kh, sq.ctx + j, sq.total, l, x);
#pragma unroll
        for (uint32_t i = 0; i < DPL; ++i) o[i] = l == 0.0f ? 0.0f : __fdiv_rn(x[i], l);
    }
#pragma unroll
    for (uint32_t i = 0; i < DPL; ++i)
        if (lane + 64u * i < p.hd) store_act_rt(p.out, at + lane + 64u * i, o[i], p.afmt);
}

// f(kernel, dynamic LDS, workgroups of it that the device holds at a time) for a head size and format.
// What a CU holds is asked once a kernel: it is the same on every device that the code is built for.
template <typename F>
int split_kernel(opure_dev* dev, uint32_t afmt, uint32_t hd, bool two, bool once, bool pieces, F&& f)
{
    auto one = [&](auto af, auto h, auto nt, auto alone, auto pc) {
        constexpr int AF = decltype(af)::value, HD = decltype(h)::value, NT = decltype(nt)::value;
        constexpr bool ONCE = decltype(alone)::value, PIECES = decltype(pc)::value;
        static std::atomic<uint64_t> done{0};
        static std::atomic<int> a_cu{0};
        auto* kernel = &k_kv4_split<AF, HD, NT, ONCE, PIECES>;
        const int rc = win_lds(dev, reinterpret_cast<const void*>(kernel), wave_lds<HD, NT, 4u>(), done);
        if (rc) return rc;
        int n = a_cu.load(std::memory_order_relaxed);
        if (n == 0)
        {
            OPURE_HIP_TRY(hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, wave_lds<HD, NT, 4u>()));
            n = std::max(n, 1);
            a_cu.store(n, std::memory_order_relaxed);
        }
        return f(kernel, wave_lds<HD, NT, 4u>(), static_cast<uint32_t>(n) * (dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u));
    };
    typedef std::integral_constant<int, 1> One;
    auto by_head = [&](auto af) {
        return win_by_head(hd, [&](auto h) {
            if constexpr (decltype(h)::value <= 128)
            {
                if (two) return one(af, h, std::integral_constant<int, 2>{}, std::false_type{}, std::false_type{});
            }
            else if (!once) return one(af, h, One{}, std::false_type{}, std::false_type{});
            return pieces ? one(af, h, One{}, std::true_type{}, std::true_type{}) : one(af, h, One{}, std::true_type{}, std::false_type{});
        });
    };
    return afmt == OPURE_A_F32   ? by_head(std::integral_constant<int, OPURE_A_F32>{})
           : afmt == OPURE_A_F16 ? by_head(std::integral_constant<int, OPURE_A_F16>{})
                                 : by_head(std::integral_constant<int, OPURE_A_BF16>{});
}

// How a call is split, and its workspace.
struct Kv4Plan {
    uint32_t tiles = 0, blocks = 0, block_rows = 0, parts = 0, least = 1;
    bool two = false, many = false;                      // blocks of 32 query rows, of 128
    bool one = false, pieces = false;                    // a workgroup a block; pieces of one size
    uint64_t acc = 0, ml = 0;                            // bytes
    uint64_t bytes() const { return acc + ml; }
};

// workspace of `slots` parts' outputs, and what a launch of `wgs` workgroups can have
int kv4_slots(const opure_attn_kv4_args* a, uint64_t slots, uint64_t wgs, uint64_t rows, Kv4Plan& w, uint32_t threads = 256u)
{
    w.acc = opure_hip::align_up(slots * w.block_rows * a->model->head_dim * 4u, 256);
    w.ml = opure_hip::align_up(slots * w.block_rows * 8u, 256);
    // a launch's threads stay in 32 bits (the join's workgroups, of 256, have a row at least)
    OPURE_REQUIRE(wgs * threads < 1ull << 32 && rows < 1u << 24, OPURE_E_CAPACITY, "4-bit attention: %u x %u rows of %u heads over max_ctx %u: too many workgroups",
                  a->batch, a->rows, a->model->n_heads, a->max_ctx);
    return OPURE_OK;
}

// Which kernels take a call, by what each would take (us; measured on 8 KV heads of 64, 80 and 128 channels, 4 of 256,
// 4 to 32 query rows each, 1 to 32 sequences of 100 to 8,000 positions; fp16 and bf16 but where fp32 is named):
//   k_kv4_one walks a sequence's tiles in one workgroup: 4.7 + channels / 150 and 0.05 a query row, and for each W tiles
//     0.4 + channels / 85 (blocks of 32 rows 1.75; 16 waves 2.2; fp32 past 192 channels, whose waves are a few registers
//     short, half as much again: 256 channels over 300 positions in 12 sequences 16.4, split 11.9), times the workgroups a CU;
//   k_kv4_split + k_kv4_join: 7.2 + channels / 100 and 0.06 a query row, 0.9 ns a tile, block of rows and 100 channels
//     (1.6 of 32 rows), and for the join 0.33 ns a query row.  Tiles are the blocks' mean.
// Measured, one / split: one row of 64 channels over 300 positions 6.0 / 8.2, 700 7.3 / 7.8, 2,000 13.4 / 7.8; of 128 over
// 300 7.1 / 8.3, 700 10.5 / 9.0; 32 sequences of 1,000 positions 10.0 / 13.7 (64 channels), 14.8 / 17.5 (128); 410 rows
// of 64 heads of 16 over themselves 13.2 / 21.8.
//   k_kv4_rows makes a tile's values once for 128 query rows, but is four waves where the others are many: from 12,000 tiles
// and blocks of 32 rows of 64 query rows or more on, past 128 channels, where its waves have a SIMD each, of 1,024.  Rows /
// split: 256 query rows of 8 KV heads of 128 channels over 500 positions 15.9 / 11.9, over 8,000 35.1 / 41.0; 64 over 8,000
// in 8 sequences 54.2 / 64.0; of 192 channels 256 over 8,000 62.1 / 60.3, 2,800 over themselves 45.7 / 65.9.
void kv4_choose(const opure_attn_kv4_args* a, uint32_t Gq, uint64_t cu, Kv4Plan& w)
{
    const double hd = a->model->head_dim, heads = static_cast<double>(a->batch) * a->model->n_kv_heads, groups = heads * w.blocks;
    w.many = Gq >= (hd <= 128.0 ? 64u : 1024u) && heads * ((Gq + 31u) / 32u) * w.tiles >= 12000.0;
    const uint32_t waves = kv4_one_waves(a->model->head_dim, w.two);
    const double wide = a->model->afmt == OPURE_A_F32 && hd > 192.0 ? 1.5 : 1.0;
    const double turn = w.two ? 1.75 : waves == 16u ? 2.2 : wide * (0.4 + hd / 85.0), rows = std::min(Gq, 32u);
    // tiles of a block: a prompt's first ones see less
    const double mean = std::min<double>(w.tiles, (a->max_ctx - a->rows / 2u) / 32u + 1u);
    const double one = 4.7 + hd / 150.0 + 0.05 * rows + turn / waves * std::max<double>(w.tiles, mean * groups / static_cast<double>(cu));
    const double split = 7.2 + hd / 100.0 + 0.06 * rows + groups * mean * hd * (w.two ? 1.6e-5 : 0.9e-5) + 3.3e-4 * heads * Gq;
    // (past 64 tiles a long sequence among short ones is what such a call waits for)
    w.one = !w.many && w.tiles <= 64u && one < split;
}

int kv4_plan(opure_dev* dev, const opure_attn_kv4_args* a, Kv4Plan& w)
{
    const opure_model* m = a->model;
    const uint32_t Gq = m->n_heads / m->n_kv_heads * a->rows;
    const uint64_t heads = static_cast<uint64_t>(a->batch) * m->n_kv_heads, rows = heads * Gq;
    const uint64_t cu = dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u;
    w.two = Gq > 16u && m->head_dim <= 128u;
    w.blocks = (Gq + (w.two ? 31u : 15u)) / (w.two ? 32u : 16u);
    w.block_rows = std::min(Gq, w.two ? 32u : 16u);
    // tiles of any block of rows: its sinks', then the window's and the rows', which begin anywhere in a tile
    const uint32_t G = m->n_heads / m->n_kv_heads, seen = std::min(a->rows, (w.block_rows + G - 2u) / G + 1u);
    const uint64_t all = (a->max_ctx + 31u) / 32u, window = a->window ? a->window : 0x7FFFFFFFu;
    w.tiles = static_cast<uint32_t>(std::min<uint64_t>(all, (a->sinks + 31ull) / 32u + (window + seen + 30ull) / 32u + 1u));
    const uint64_t groups = heads * w.blocks;
    kv4_choose(a, Gq, cu, w);
    const uint32_t asked = dev->kv4_kernels;
    if (asked != OPURE_KV4_BEST)
    {
        w.many = asked == OPURE_KV4_ROWS;
        w.one = asked == OPURE_KV4_ONE;
        OPURE_REQUIRE(asked != OPURE_KV4_PIECES || (w.blocks == 1u && !w.two), OPURE_E_UNSUPPORTED,
                      "4-bit attention: pieces of one size have up to 16 query rows a KV head, not %u", Gq);
    }
    if (w.many)
    {
        w.blocks = (Gq + ROWS_BLOCK - 1u) / ROWS_BLOCK;
        w.block_rows = std::min(Gq, ROWS_BLOCK);
        // Two workgroups a CU; but one part, and no join, where a short walk takes half the CUs as it is (779 rows of 24 heads of
        // 112 over themselves 24.2 us, in three parts 30.4; 1,500 of 16 of 192 over 1,000 and themselves 167 and 131)
        const uint64_t fill = 2u * heads * w.blocks >= cu && w.tiles <= 32u ? 1u : std::max<uint64_t>(1u, 2u * cu / (heads * w.blocks));
        w.parts = static_cast<uint32_t>(std::min<uint64_t>(fill, std::min((w.tiles + 7u) / 8u, MAX_PARTS)));
        const uint64_t wgs = heads * w.blocks * w.parts;
        return kv4_slots(a, w.parts == 1u ? 0u : wgs, wgs, rows, w);
    }
    if (w.one)
    {
        w.parts = 1u;
        return kv4_slots(a, 0u, groups, rows, w, 64u * kv4_one_waves(m->head_dim, w.two));
    }
    uint32_t room = 0;
    auto holds = [&](auto, uint32_t, uint32_t n) {
        room = n;
        return OPURE_OK;
    };
    if (w.blocks == 1u && (a->batch > 1u || asked == OPURE_KV4_PIECES))
    {
        int rc = split_kernel(dev, m->afmt, m->head_dim, w.two, true, true, holds);
        if (rc) return rc;
        const uint64_t hold = std::max<uint64_t>(1u, room / m->n_kv_heads), all = static_cast<uint64_t>(a->batch) * w.tiles;
        w.pieces = asked == OPURE_KV4_BEST ? !w.two && all >= 32u * hold : asked == OPURE_KV4_PIECES;
        if (w.pieces)
        {
            // the sum of the sequences' tiles stays in 31 bits
            OPURE_REQUIRE(all < 1u << 31, OPURE_E_CAPACITY, "4-bit attention: %u sequences of max_ctx %u", a->batch, a->max_ctx);
            w.least = 4u;
            w.parts = static_cast<uint32_t>(hold);
            return kv4_slots(a, (hold + a->batch - 1u) * m->n_kv_heads, hold * m->n_kv_heads, rows, w);
        }
    }
    const int rc = split_kernel(dev, m->afmt, m->head_dim, w.two, w.blocks == 1u, false, holds);
    if (rc) return rc;
    // Parts of a group: as many as the device holds at a time, each of at least four tiles (one a wave), or of so many
    // that the part's outputs, written and read again, stay a quarter of its keys and values; three times as many where
    // a wave still has four tiles, which evens out ragged sequences
    const uint32_t least = std::max(4u, w.block_rows / 4u);
    const uint64_t fill = std::max<uint64_t>(1u, room / groups), more = std::min<uint64_t>(3ull * room / groups, w.tiles / 16u);
    w.parts = static_cast<uint32_t>(std::min<uint64_t>(std::max(fill, more), std::min((w.tiles + least - 1u) / least, MAX_PARTS)));
    return kv4_slots(a, groups * w.parts, groups * w.parts, rows, w);
}

int kv4_validate(const opure_attn_kv4_args* a)
{
    OPURE_REQUIRE(a && a->model && a->kv && a->kv->pool && a->kv->page_table, OPURE_E_INVALID, "4-bit attention: null argument, model or cache");
    const opure_model* m = a->model;
    const opure_kv* kv = a->kv;
    OPURE_REQUIRE(m->n_kv_heads >= 1 && m->n_heads >= 1 && m->n_heads % m->n_kv_heads == 0, OPURE_E_INVALID,
                  "4-bit attention: n_heads %u %% n_kv_heads %u != 0", m->n_heads, m->n_kv_heads);
    OPURE_REQUIRE(m->head_dim >= 16 && m->head_dim <= 256 && m->head_dim % 16 == 0, OPURE_E_UNSUPPORTED,
                  "4-bit attention: head_dim %u not in 16..256 step 16", m->head_dim);
    OPURE_REQUIRE(m->afmt <= OPURE_A_BF16, OPURE_E_INVALID, "4-bit attention: bad activation format");
    OPURE_REQUIRE(kv->page_size == OPURE_PAGE_SIZE, OPURE_E_UNSUPPORTED, "4-bit attention: page_size must be %d", OPURE_PAGE_SIZE);
    OPURE_REQUIRE(kv->n_pages >= 1 && kv->max_pages_per_seq >= 1, OPURE_E_INVALID, "4-bit attention: the cache has no pages");
    OPURE_REQUIRE(a->layer < m->n_layers, OPURE_E_INVALID, "4-bit attention: layer %u of %u", a->layer, m->n_layers);
    OPURE_REQUIRE(a->batch >= 1 && a->batch <= OPURE_MAX_BATCH_ROWS && a->rows >= 1 && a->rows <= OPURE_MAX_PROMPT_ROWS, OPURE_E_CAPACITY,
                  "4-bit attention: %u rows x %u sequences outside 1..%d x 1..%d", a->rows, a->batch, OPURE_MAX_PROMPT_ROWS, OPURE_MAX_BATCH_ROWS);
    // the query rows' indexes stay in 32 bits, and a page's bytes
    OPURE_REQUIRE(static_cast<uint64_t>(m->n_heads) * a->batch * a->rows <= 1u << 25 && m->n_kv_heads <= 1u << 18, OPURE_E_CAPACITY,
                  "4-bit attention: %u x %u rows of %u heads", a->batch, a->rows, m->n_heads);
    const uint64_t slots = static_cast<uint64_t>(kv->max_pages_per_seq) * OPURE_PAGE_SIZE;
    OPURE_REQUIRE(a->max_ctx >= a->rows && a->max_ctx <= slots && a->max_ctx <= 0x7FFFFFFFu - OPURE_MAX_PROMPT_ROWS, OPURE_E_CAPACITY,
                  "4-bit attention: max_ctx %u below %u rows or beyond the page table's %llu", a->max_ctx, a->rows, (unsigned long long)slots);
    OPURE_REQUIRE(a->sinks <= 0x7FFFFFFFu, OPURE_E_INVALID, "4-bit attention: %u sinks", a->sinks);
    OPURE_REQUIRE((reinterpret_cast<uintptr_t>(kv->pool) & 15u) == 0u && (reinterpret_cast<uintptr_t>(kv->page_table) & 3u) == 0u,
                  OPURE_E_INVALID, "4-bit attention: pool must be 16-byte aligned, page_table 4-byte");
    return OPURE_OK;
}

}  // namespace

using namespace opure_hip;

extern "C" int opure_attn_kv4_reserve(opure_dev* dev, const opure_attn_kv4_args* a)
{
    OPURE_REQUIRE(dev, OPURE_E_INVALID, "opure_attn_kv4_reserve: null device");
    const int rc = kv4_validate(a);
    if (rc) return rc;
    const DeviceGuard on(dev);
    Kv4Plan w;
    const int rp = kv4_plan(dev, a, w);
    return rp ? rp : ensure_workspace(dev, w.bytes());
}

extern "C" int opure_debug_kv4_kernels(opure_dev* dev, const opure_attn_kv4_args* a, uint32_t* kernels, uint32_t* parts)
{
    OPURE_REQUIRE(dev && kernels && parts, OPURE_E_INVALID, "opure_debug_kv4_kernels: null argument");
    const int rc = kv4_validate(a);
    if (rc) return rc;
    const DeviceGuard on(dev);
    Kv4Plan w;
    const int rp = kv4_plan(dev, a, w);
    if (rp) return rp;
    *kernels = w.many ? OPURE_KV4_ROWS : w.one ? OPURE_KV4_ONE : w.pieces ? OPURE_KV4_PIECES : OPURE_KV4_SPLIT;
    *parts = w.parts;
    return OPURE_OK;
}

extern "C" int opure_attn_kv4_paged(opure_dev* dev, const opure_attn_kv4_args* a)
{
    OPURE_REQUIRE(dev && a && a->q && a->out && a->seq_len, OPURE_E_INVALID, "opure_attn_kv4_paged: null argument");
    int rc = kv4_validate(a);
    if (rc) return rc;
    OPURE_REQUIRE((reinterpret_cast<uintptr_t>(a->q) & 15u) == 0u && (reinterpret_cast<uintptr_t>(a->out) & 7u) == 0u &&
                      (reinterpret_cast<uintptr_t>(a->seq_len) & 3u) == 0u,
                  OPURE_E_INVALID, "opure_attn_kv4_paged: q must be 16-byte aligned, out 8-byte, seq_len 4-byte");
    const opure_model* m = a->model;
    const uint64_t bytes = static_cast<uint64_t>(a->batch) * a->rows * m->n_heads * m->head_dim * act_bytes(m->afmt);
    OPURE_REQUIRE(!overlaps(a->out, bytes, a->q, bytes), OPURE_E_INVALID, "opure_attn_kv4_paged: out overlaps q");
    OPURE_REQUIRE(!overlaps(a->out, bytes, a->kv->pool, kv_pool_bytes(m, OPURE_KV_I4, a->kv->n_pages)) &&
                      !overlaps(a->out, bytes, a->kv->page_table, static_cast<uint64_t>(a->batch) * a->kv->max_pages_per_seq * 4u) &&
                      !overlaps(a->out, bytes, a->seq_len, a->batch * 4u), OPURE_E_INVALID, "opure_attn_kv4_paged: out overlaps the cache");
    // the call's parts go to the workspace, which may also move
    OPURE_REQUIRE(!overlaps(dev->ws, dev->ws_bytes, a->q, bytes) && !overlaps(dev->ws, dev->ws_bytes, a->out, bytes), OPURE_E_INVALID,
                  "opure_attn_kv4_paged: q or out in the device's workspace");
    const DeviceGuard on(dev);
    Kv4Plan w;
    rc = kv4_plan(dev, a, w);
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
    p.n_heads = m->n_heads;
    p.n_kv = m->n_kv_heads;
    p.hd = m->head_dim;
    p.rows = a->rows;
    p.n_pages = a->kv->n_pages;
    p.max_pages = a->kv->max_pages_per_seq;
    p.layer = a->layer;
    p.afmt = m->afmt;
    p.window = a->window == 0u || a->window > 0x7FFFFFFFu ? 0x7FFFFFFFu : a->window;
    p.sinks = a->sinks;
    p.cap = a->max_ctx;
    p.scale = m->attn_scale;
    p.err = dev->err;
    p.parts = w.parts;
    p.blocks = w.blocks;
    p.block_rows = w.block_rows;
    p.two = w.many ? 2u : w.two ? 1u : 0u;
    p.tiles = w.tiles;
    p.combine_rows = a->batch * a->rows * p.n_heads;
    p.least = w.least;
    p.pieces = w.pieces ? 1u : 0u;
    p.by_parts = w.parts > 1u ? static_cast<uint32_t>(((1ull << 32) + w.parts - 1u) / w.parts) : 0u;
    p.batch = a->batch;
    const uint32_t wgs = p.n_kv * w.parts * (w.pieces ? 1u : w.blocks * a->batch);
    auto launch = [&](auto kernel, uint32_t lds, uint32_t = 0) {
        OPURE_LAUNCH(dev, kernel, dim3(wgs), dim3(256), lds, p);
        OPURE_LAUNCH_CHECK("4-bit attention");
        return OPURE_OK;
    };
    if (w.one) return kv4_one_launch(dev, p, wgs);
    rc = w.many ? kv4_rows_launch(dev, p, wgs) : split_kernel(dev, p.afmt, p.hd, w.two, w.blocks == 1u, w.pieces, launch);
    if (rc || (w.many && w.parts == 1u)) return rc;
    const bool wide = w.parts > (w.pieces ? 8u * a->batch : 8u);
    p.combine_wgs = wide ? p.combine_rows : (p.combine_rows + 3u) / 4u;
    auto join = [&](auto all) {
        constexpr bool WIDE = decltype(all)::value;
        const dim3 grid(p.combine_wgs), block(256);
        switch ((p.hd + 63u) / 64u)
        {
        case 1: OPURE_LAUNCH(dev, (k_kv4_join<WIDE, 1>), grid, block, 0, p); break;
        case 2: OPURE_LAUNCH(dev, (k_kv4_join<WIDE, 2>), grid, block, 0, p); break;
        case 3: OPURE_LAUNCH(dev, (k_kv4_join<WIDE, 3>), grid, block, 0, p); break;
        default: OPURE_LAUNCH(dev, (k_kv4_join<WIDE, 4>), grid, block, 0, p); break;
        }
    };
    if (wide) join(std::true_type{});
    else join(std::false_type{});
    OPURE_LAUNCH_CHECK("k_kv4_join");
    return OPURE_OK;
}
