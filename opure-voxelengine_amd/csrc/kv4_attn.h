// ============================================================================
//  kv4_attn.h -- what the kernels of attention over the 4-bit cache share.
// ============================================================================
#pragma once
#include "kv4.h"
#include "window.h"

#include <algorithm>

namespace opure_kv4 {

using namespace opure_win;

constexpr uint32_t MAX_PARTS = 64;                         // of a (sequence, KV head, block of query rows): a lane of the joining wave each
constexpr float LOG2E = 1.44269504088896340736f;
// With the products s of a row and c = scale log2 e, weights are 2^(s c - M) by one fused multiply-add, M the largest
// s c rounded down to a whole number: M, what it is told apart by and 2^(M - M') are exact, so a weight is off by its
// exponent's own rounding alone, however large the scores.  (With M = m c rounded, the rounding, 2^5 at 2^29, stood in
// every weight's exponent.)  A row is scaled to a new M only where s c passes the old one by LAG.  Weights are held
// times 2^SHIFT, so the largest of 2^15 is still in fp16, and what fp16 loses at its small end lies 2^36 below 1.  Past
// FAR, where SHIFT - M would be rounded in the end, a row's sum is NaN, and it is computed position by position.
constexpr float SHIFT = 12.0f, LAG = 3.0f, FAR = 0x1p22f;
__device__ __forceinline__ bool has_grown(float m, float mx, float c) { return m == NEG_INF ? mx > NEG_INF : __fmaf_rn(mx, c, -m) > LAG; }
// m, and the row's sum l, to a new maximum mx where it has grown; returns the factor of what is there already
__device__ __forceinline__ float grow(bool grown, float mx, float c, float& m, float& l)
{
    const float to = grown ? __builtin_floorf(__fmul_rn(mx, c)) : m, a = m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(__fsub_rn(m, to));
    m = to;
    // a NaN whose bits an instruction has room for: another one takes two registers, and a workgroup a CU of three kernels (96 channels 8.3 us, so 10.6)
    l = grown && !(__builtin_fabsf(to) <= FAR) ? __uint_as_float(0xFFFFFFFFu) : __fmul_rn(l, a);
    return a;
}

typedef u4v u4a __attribute__((aligned(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef u2v u2a __attribute__((aligned(4)));

// N consecutive words, 4-byte aligned
template <uint32_t N, bool ONCE>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t (&w)[N])
{
    constexpr uint32_t Q = N / 4u * 4u;
#pragma unroll
    for (uint32_t i = 0; i < Q; i += 4u)
    {
        const u4a* q = reinterpret_cast<const u4a*>(p + i);
        u4v v;
        if constexpr (ONCE) v = __builtin_nontemporal_load(q);
        else v = *q;
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x) w[i + x] = v[x];
    }
    if constexpr ((N & 2u) != 0u)
    {
        const u2a* q = reinterpret_cast<const u2a*>(p + Q);
        u2v v;
        if constexpr (ONCE) v = __builtin_nontemporal_load(q);
        else v = *q;
        w[Q] = v[0];
        w[Q + 1u] = v[1];
    }
    if constexpr ((N & 1u) != 0u)
    {
        if constexpr (ONCE) w[N - 1u] = __builtin_nontemporal_load(p + N - 1u);
        else w[N - 1u] = p[N - 1u];
    }
}

// Two pages of a KV head, positions 16 x + 0..15 of page x: lane (r, g) has K codes
// of token r and channels 8 g of each group, and V codes of channels r and 16 + r of
// each group and the tokens 4 g .. 4 g + 3.
template <int HD, bool ONCE>
struct Kv4Tile {
    static constexpr uint32_t NG = groups(HD);
    uint32_t kw[2][NG], ks[2][NG], vw[2][NG];
    u4v vs[2][NG];                                         // [scale 0 1, scale 2 3, base 0 1, base 2 3]
    __device__ __forceinline__ void load_k(const uint8_t* a, const uint8_t* b, uint32_t lane)
    {
#pragma unroll
        for (uint32_t x = 0; x < 2; ++x)
        {
            const uint32_t* at = reinterpret_cast<const uint32_t*>(x ? b : a);
            load_words<NG, ONCE>(at + lane * NG, kw[x]);
            load_words<NG, ONCE>(at + k_scales(NG) / 4u + (lane & 15u) * NG, ks[x]);
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t* a, const uint8_t* b, uint32_t lane)
    {
#pragma unroll
        for (uint32_t x = 0; x < 2; ++x)
        {
            const uint8_t* at = x ? b : a;
            load_words<NG, ONCE>(reinterpret_cast<const uint32_t*>(at + v_codes(NG)) + lane * NG, vw[x]);
#pragma unroll
            for (uint32_t p = 0; p < NG; ++p) vs[x][p] = win_load<ONCE>(at + v_scales(NG) + ((lane >> 4) * NG + p) * 16u);
        }
    }
    // group p of page x as fp16 numbers
    __device__ __forceinline__ u4v k(const Bits& bits, uint32_t x, uint32_t p) const
    {
        const half2_t sb = pair(ks[x][p]), s = {sb[0], sb[0]}, b = {sb[1], sb[1]};
        const uint32_t w = kw[x][p];
        return u4v{values(bits.codes<0>(w), s, b), values(bits.codes<1>(w), s, b), values(bits.codes<2>(w), s, b), values(bits.codes<3>(w), s, b)};
    }
    // channels 32 p + 16 T + r of both pages' tokens
    template <int T>
    __device__ __forceinline__ u4v v(const Bits& bits, uint32_t p) const
    {
        u4v o;
#pragma unroll
        for (uint32_t x = 0; x < 2; ++x)
        {
            o[2 * x] = values(bits.template codes<2 * T>(vw[x][p]), pair(vs[x][p][0]), pair(vs[x][p][2]));
            o[2 * x + 1] = values(bits.template codes<2 * T + 1>(vw[x][p]), pair(vs[x][p][1]), pair(vs[x][p][3]));
        }
        return o;
    }
};

__device__ __forceinline__ f4_t mfma(u4v a, u4v b, f4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// A number worked out from all results of a run of matrix instructions, in the block
// that asked for them: whoever reads them behind a branch finds them written.  (The
// compiler spaces a read and its matrix instruction by the longest way through the
// blocks between them, and a short way then reads what was there before.)
__device__ __forceinline__ float settled(float v)
{
    asm volatile("" : "+v"(v));
    return v;
}
// The same after a loop of them: as many clocks as the longest takes.
__device__ __forceinline__ void settle()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
}

// A query row in fp16: of an fp16 model as it is, else times the power of two that
// puts its largest magnitude just below 2^9 (bf16's 8 bits fit, and what fp16 cannot
// hold of its small numbers is 2^-34 of the largest); an fp32 row is the sum of two.
// A lane takes 8 channels of each step of W = 8 PARTS channels, the `part`-th.  Returns
// the factor of its scores in powers of two.
template <int AF, int HD, uint32_t PARTS>
__device__ __forceinline__ float load_query(const WinParams& p, uint64_t row, uint32_t part,
                                            u4v (&q)[AF == OPURE_A_F32 ? 2 : 1][(HD + 8u * PARTS - 1u) / (8u * PARTS)])
{
    constexpr uint32_t W = 8u * PARTS, STEPS = (HD + W - 1u) / W;
    const float c = __fmul_rn(p.scale, LOG2E);
    auto there = [&](uint32_t s) { return (s + 1u) * W <= HD || s * W + 8u * part < HD; };
    if constexpr (AF == OPURE_A_F16)
    {
        const uint8_t* at = static_cast<const uint8_t*>(p.q) + row * (HD * 2u) + 16u * part;
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s) q[0][s] = there(s) ? *reinterpret_cast<const u4v*>(at + 2u * W * s) : u4v{0u, 0u, 0u, 0u};
        return c;
    }
    else
    {
        float x[STEPS][8], top = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s)
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
            {
                x[s][i] = there(s) ? load_act<AF>(p.q, row * HD + W * s + 8u * part + i) : 0.0f;
                top = fmaxf(top, __builtin_fabsf(x[s][i]));
            }
        if (__any(top == __builtin_huge_valf()))           // infinities do not count
        {
            top = 0.0f;
#pragma unroll
            for (uint32_t s = 0; s < STEPS; ++s)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) top = fmaxf(top, __builtin_isfinite(x[s][i]) ? __builtin_fabsf(x[s][i]) : 0.0f);
        }
        if constexpr (PARTS == 4u) top = max_xor16(top);
        const int e = __builtin_amdgcn_frexp_expf(max_xor32(top)) - 9;
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
            {
                const float y0 = __builtin_ldexpf(x[s][2 * i], -e), y1 = __builtin_ldexpf(x[s][2 * i + 1], -e);
                q[0][s][i] = win_pack<OPURE_A_F16>(y0, y1);
                if constexpr (AF == OPURE_A_F32)
                    q[1][s][i] = win_pack<OPURE_A_F16>(__fsub_rn(y0, win_low<OPURE_A_F16>(q[0][s][i])), __fsub_rn(y1, win_high<OPURE_A_F16>(q[0][s][i])));
            }
        return __builtin_ldexpf(c, e);
    }
}

// Scores in powers of two are c >= 0 times the products: the scale's sign goes to the query.
template <int AF, int HD, uint32_t PARTS, uint32_t QT, uint32_t STEPS>
__device__ __forceinline__ float signed_query(const WinParams& p, uint64_t row, uint32_t part, u4v (&q)[QT][STEPS])
{
    const float c = load_query<AF, HD, PARTS>(p, row, part, q);
    if (p.scale < 0.0f)
#pragma unroll
        for (uint32_t z = 0; z < QT; ++z)
#pragma unroll
            for (uint32_t s = 0; s < STEPS; ++s) q[z][s] ^= u4v{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
    return __builtin_fabsf(c);
}

// One query row by one wave, exactly as the formulas say it; a position that the
// row does not see is not read.  qs: the row in LDS (hd floats).
__device__ inline void kv4_row(const WinParams& p, const float* qs, uint32_t b, uint32_t kh, uint32_t pos, uint32_t total, float& l, float (&o)[4])
{
    const uint32_t lane = threadIdx.x & 63u, hd = p.hd, ng = groups(hd);
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    const uint8_t* pool = static_cast<const uint8_t*>(p.pool);
    const uint32_t end = min(pos + 1u, total), low = pos + 1u > p.window ? pos + 1u - p.window : 0u;
    float m = NEG_INF;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = 0.0f;
    for (uint32_t t0 = 0; t0 < end; t0 += 64u)
    {
        if (t0 >= p.sinks && t0 + 64u <= low)
        {
            t0 = low / 64u * 64u - 64u;                    // between the sinks and the window
            continue;
        }
        const uint32_t t = t0 + lane;
        const bool in = t < end && win_sees(p, pos, t);
        const int32_t pg = in ? win_page(p, pt, t) : -1;
        float s = in ? __builtin_nanf("") : NEG_INF;
        if (pg >= 0)
        {
            const uint8_t* at = pool + block_at(p.layer, p.n_pages, static_cast<uint32_t>(pg), p.n_kv, kh, ng);
            float acc = 0.0f;
            for (uint32_t d = 0; d < hd; ++d) acc = __fmaf_rn(qs[d], k_value(at, ng, t % OPURE_PAGE_SIZE, d), acc);
            s = __fmul_rn(acc, p.scale);
        }
        const float mx = fmaxf(m, wave_max64(s));          // a NaN score leaves the maximum and reaches the sum
        const float ms = mx == NEG_INF ? 0.0f : mx;
        const float a = expf_ref(__fsub_rn(m, ms)), e = in ? expf_ref(__fsub_rn(s, ms)) : 0.0f;
        m = mx;
        l = __fmaf_rn(l, a, wave_sum64(e));
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __fmul_rn(o[i], a);
        uint64_t left = __ballot(in && pg >= 0);
        while (left)
        {
            const int k = __builtin_ctzll(left);
            left &= left - 1u;
            const float w = __shfl(e, k);
            const uint32_t pk = static_cast<uint32_t>(__shfl(pg, k)), tk = t0 + static_cast<uint32_t>(k);
            const uint8_t* at = pool + block_at(p.layer, p.n_pages, pk, p.n_kv, kh, ng);
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const uint32_t d = lane + 64u * i;
                if (d < hd) o[i] = __fmaf_rn(w, v_value(at, ng, tk % OPURE_PAGE_SIZE, d), o[i]);
            }
        }
    }
}

// How the tiles are shared out: those of all sequences, one sequence's behind the
// other's, in pieces of one size, so that all workgroups that the device holds have as
// much to do whatever the lengths are.  A piece is a workgroup of each KV head and block
// of rows; it may hold the end of a sequence, whole ones and the begin of one.  Piece w's
// part of sequence b has slot w + b: going on to the next part is going on to the next
// piece or to the next sequence.
//   32 sequences of 1,024 to 16,384 positions (8 KV heads of 128): a sixth of each
// sequence a workgroup 68 us, pieces that end with their sequence 62 to 65, these 53 to 56.
struct Share {
    uint32_t size, total;                                  // tiles of a piece, of all
    uint32_t b, before;                                    // a sequence, tiles before it
};

__device__ __forceinline__ WinSpan seq_span(const WinParams& p, const WinSeq& sq) { return win_span<32u>(p, sq, sq.ctx, sq.ctx + p.rows); }

// a sequence's tiles; one at least, so that it has a part
__device__ __forceinline__ uint32_t seq_tiles(const WinParams& p, uint32_t b)
{
    const int32_t len = p.seq_len[b];
    WinSeq sq;
    sq.ctx = len < 0 ? 0u : static_cast<uint32_t>(len);
    sq.total = min(sq.ctx + p.rows, p.cap);
    return max(seq_span(p, sq).n, 1u);
}

__device__ __forceinline__ uint32_t sum_lanes(uint32_t v)
{
    v += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true));
    v += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true));
    v += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xF, 0xF, true));
    v += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xF, 0xF, true));
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 0) + __builtin_amdgcn_readlane(static_cast<int>(v), 16) +
                                 __builtin_amdgcn_readlane(static_cast<int>(v), 32) + __builtin_amdgcn_readlane(static_cast<int>(v), 48));
}

// n / p.parts, n < 2^31; of n p.parts itself n
__device__ __forceinline__ uint32_t part_of(const WinParams& p, uint32_t n) { return p.parts == 1u ? n : __umulhi(n, p.by_parts); }

// The shares, and of `u` a piece the sequence that it begins in (PIECE), else sequence u.
template <bool PIECE>
__device__ __forceinline__ Share share_out(const WinParams& p, uint32_t u)
{
    const uint32_t lane = threadIdx.x & 63u;               // has sequences 4 lane .. 4 lane + 3
    uint32_t n[4], mine = 0, most = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) n[i] = seq_tiles(p, min(4u * lane + i, p.batch - 1u));
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
    {
        most = max(most, n[i]);
        n[i] = 4u * lane + i < p.batch ? n[i] : 0u;
        mine += n[i];
    }
    // as fp32: off by 2^-24 of it, which the room for two more parts covers
    most = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(wave_max64(static_cast<float>(most)))));
    Share s;
    s.total = sum_lanes(mine);
    // a sequence's parts, one a piece that it meets, are 64 at most
    s.size = max(max(part_of(p, s.total) + 1u, most / (MAX_PARTS - 2u) + 1u), p.least);
    uint32_t before = mine;
#pragma unroll
    for (uint32_t o = 1; o < 64u; o <<= 1)
    {
        const uint32_t x = __shfl_up(before, o);
        if (lane >= o) before += x;
    }
    before -= mine;
    const uint32_t at = PIECE ? min(u * s.size, s.total - 1u) : 0u;
    const uint32_t l = PIECE ? static_cast<uint32_t>(__popcll(__ballot(before <= at && mine != 0u))) - 1u : u >> 2;
    auto of = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(l))); };
    s.b = 4u * l;
    s.before = of(before);
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
    {
        const uint32_t c = of(n[i]);
        if (s.b == 4u * l + i && (PIECE ? at >= s.before + c : (u & 3u) > i))
        {
            s.before += c;
            ++s.b;
        }
    }
    return s;
}

// The lane as a number that is new each time: what follows from it is worked out where it
// is used, not kept in registers across a loop over sequences (168 of them and spills, 142 without).
__device__ __forceinline__ uint32_t once_more(uint32_t v)
{
    asm volatile("" : "+v"(v));
    return v;
}

// A wave's run over tiles of a sequence for 16 NT query rows of a KV head (row qi = j
// group + head), every W-th of them: a running maximum, sum and output in registers.
// Lane (r, g) holds scores of query row r and the tokens 4 g .. 4 g + 3 of both pages,
// which is its operand P^T in the order that the V codes have.  Each tile's words are
// asked for when the last one's are used up.
template <int AF, int HD, int NT, bool ONCE, uint32_t W>
struct Kv4Wave {
    typedef Kv4Tile<HD, ONCE> T;
    static constexpr uint32_t TT = 32u, DT = HD / 16u, NG = T::NG, QT = AF == OPURE_A_F32 ? 2u : 1u;
    // a weight's rounding rest counts: bf16 results are rounded 2^3 more coarsely than a weight (with it their error is 1.66e-3
    // for 1.67e-3, and a prompt of 2,048 rows over 6,000 takes 357 us for 276, a long batch of single rows 54.7 for 52.6)
    static constexpr bool REST = AF != OPURE_A_BF16;
    const WinParams& p;
    const Bits bits;
    uint32_t lane, g, r;
    const uint32_t G, Gq, kh, q0, j0, j1, page_bytes;      // j0, j1: the block's first and last row
    const uint8_t* const base;
    // the sequence, the wave's tiles i, i + W, .. below last of its list, its queries and first words
    const int32_t* pt;
    WinSeq sq;
    WinSpan span;
    u4v q[NT][QT][NG];
    uint32_t jr[NT], i, last;
    float c[NT];
    int32_t e = -1, pa = -1, pb = -1;
    T tl;
    // a row's M, this lane's share of its sum, its output
    f4_t o[DT][NT];
    float m[NT], l[NT];

    __device__ __forceinline__ Kv4Wave(const WinParams& params, uint32_t head, uint32_t first_row)
        : p(params), G(params.n_heads / params.n_kv), Gq(G * params.rows), kh(head), q0(first_row),
          j0(first_row / G), j1(min(first_row + 16u * NT - 1u, Gq - 1u) / G), page_bytes(params.n_kv * (BLOCK * NG)),
          base(static_cast<const uint8_t*>(params.pool) + block_at(params.layer, params.n_pages, 0u, params.n_kv, head, NG))
    {
    }
    // pages of tile i of the list: -1 past the sequence, missing or not in the pool
    __device__ __forceinline__ int32_t entry(uint32_t x) const { return pt[min(span.tile(min(x, span.n - 1u)) * 2u + (lane & 1u), p.max_pages - 1u)]; }
    __device__ __forceinline__ int32_t page(int32_t es, uint32_t x, uint32_t which) const
    {
        const int32_t pg = __builtin_amdgcn_readlane(es, which);
        return (span.tile(x) * 2u + which) * OPURE_PAGE_SIZE < sq.total && static_cast<uint32_t>(pg) < p.n_pages ? pg : -1;
    }
    __device__ __forceinline__ const uint8_t* at(int32_t pg) const
    {
        return base + static_cast<uint64_t>(pg < 0 ? 0u : static_cast<uint32_t>(pg)) * page_bytes;
    }
    __device__ __forceinline__ void seek(uint32_t b)
    {
        lane = once_more(threadIdx.x & 63u);
        g = lane >> 4;
        r = lane & 15u;
        pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
        sq = win_seq(p, p.seq_len[b]);
        // what the block's rows see (of all rows: 859 of 8 heads of 192 behind a window of 96 34.7 us, so 18.3)
        span = win_span<TT>(p, sq, sq.ctx + j0, sq.ctx + j1 + 1u);
    }
    // tiles first .. end - 1 of the list, the wave's from `mine` on
    __device__ __forceinline__ void start(uint32_t b, uint32_t mine, uint32_t end)
    {
        i = mine;
        last = end;
        if (i < last)
        {
            e = entry(i);
            pa = page(e, i, 0u);
            pb = page(e, i, 1u);
            tl.load_k(at(pa), at(pb), lane);
            e = entry(i + W);
        }
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
        {
            const uint32_t qi = min(q0 + 16u * n + r, Gq - 1u);
            jr[n] = qi / G;
            c[n] = signed_query<AF, HD, 4>(p, (static_cast<uint64_t>(b) * p.rows + jr[n]) * p.n_heads + kh * G + (qi - jr[n] * G), g, q[n]);
        }
    }
    __device__ __forceinline__ void run()
    {
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
        {
            m[n] = NEG_INF;
            l[n] = 0.0f;
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) o[d][n] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        if (i >= last) return;
        tl.load_v(at(pa), at(pb), lane);                   // not before: with the values' words over a merge 168 registers are not enough
        while (true)
        {
            const uint32_t t0 = span.tile(i) * TT;
            const bool more = i + W < last;
            const int32_t na = more ? page(e, i + W, 0u) : pa, nb = more ? page(e, i + W, 1u) : pb;
            if (more) e = entry(i + 2u * W);
            if (pa < 0 || pb < 0)
            {
                // positions without a page: NaN keys for the rows that see them
#pragma unroll
                for (uint32_t s = 0; s < NG; ++s)
                {
                    tl.ks[0][s] = pa < 0 ? 0x7E007E00u : tl.ks[0][s];
                    tl.ks[1][s] = pb < 0 ? 0x7E007E00u : tl.ks[1][s];
                }
            }
            f4_t acc[2][NT];
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n) acc[x][n] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t s = 0; s < NG; ++s)
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x)
                {
                    const u4v k = tl.k(bits, x, s);
#pragma unroll
                    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                        for (uint32_t z = 0; z < QT; ++z) acc[x][n] = mfma(k, q[n][z][s], acc[x][n]);
                }
            if (more) tl.load_k(at(na), at(nb), lane);
            // every row sees every position
            const bool full = t0 + TT <= min(sq.ctx + j0 + 1u, sq.total) && (t0 + TT <= p.sinks || t0 + p.window > sq.ctx + j1);
            u4v hi[NT], lo[NT];
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
            {
                float s[8];
#pragma unroll
                for (uint32_t y = 0; y < 8; ++y) s[y] = acc[y >> 2][n][y & 3u];
                auto largest = [&]() {
                    float v = s[0];
#pragma unroll
                    for (uint32_t y = 1; y < 8; ++y) v = fmaxf(v, s[y]);
                    return v;
                };
                float mx = settled(largest());
                if (!full)
                {
                    const WinMask mask(p, sq.ctx + jr[n], sq.total, t0 + 4u * g);
#pragma unroll
                    for (uint32_t y = 0; y < 8; ++y) s[y] = mask.sees(static_cast<int32_t>(16u * (y >> 2) + (y & 3u))) ? s[y] : NEG_INF;
                    mx = largest();
                }
                mx = max_xor32(max_xor16(mx));
                const bool grown = has_grown(m[n], mx, c[n]);
                if (__any(grown))
                {
                    const float a = grow(grown, mx, c[n], m[n], l[n]);
#pragma unroll
                    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
                        for (uint32_t y = 0; y < 4; ++y) o[d][n][y] = __fmul_rn(o[d][n][y], a);
                }
                const float down = m[n] == NEG_INF ? 0.0f : __fsub_rn(SHIFT, m[n]);
#pragma unroll
                for (uint32_t y = 0; y < 8; ++y)
                {
                    s[y] = __builtin_amdgcn_exp2f(__fmaf_rn(s[y], c[n], down));
                    l[n] += s[y];                              // this lane's share of the row's sum
                }
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y)
                {
                    hi[n][y] = win_pack<OPURE_A_F16>(s[2 * y], s[2 * y + 1]);
                    if constexpr (REST)
                        lo[n][y] = win_pack<OPURE_A_F16>(__fsub_rn(s[2 * y], win_low<OPURE_A_F16>(hi[n][y])), __fsub_rn(s[2 * y + 1], win_high<OPURE_A_F16>(hi[n][y])));
                }
            }
            if (t0 + TT > sq.total || pa < 0 || pb < 0)
            {
                // slots past the sequence and pages that are not there hold anything: 0
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x)
                {
                    const uint32_t t = t0 + 16u * x + 4u * g, n = (x ? pb : pa) < 0 || t >= sq.total ? 0u : min(sq.total - t, 4u);
                    const uint32_t m0 = n >= 2u ? 0xFFFFFFFFu : n == 1u ? 0xFFFFu : 0u, m1 = n >= 4u ? 0xFFFFFFFFu : n == 3u ? 0xFFFFu : 0u;
#pragma unroll
                    for (uint32_t s = 0; s < NG; ++s) tl.vs[x][s] &= u4v{m0, m1, m0, m1};
                }
            }
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d)
            {
                const u4v v = d & 1u ? tl.template v<1>(bits, d >> 1) : tl.template v<0>(bits, d >> 1);
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n)
                {
                    if constexpr (REST) o[d][n] = mfma(v, lo[n], o[d][n]);
                    o[d][n] = mfma(v, hi[n], o[d][n]);
                }
            }
            if (!more) break;
            tl.load_v(at(na), at(nb), lane);
            pa = na;
            pb = nb;
            i += W;
        }
        settle();
    }
    // to LDS for the workgroup's merge: acc [wave][DT][NT][64], ml [wave][NT][16][2]
    __device__ __forceinline__ void leave(uint32_t wave, f4_t* acc, float* ml)
    {
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
        {
            l[n] = add_xor32(add_xor16(l[n]));
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) acc[((wave * DT + d) * NT + n) * 64u + lane] = o[d][n];
            if (g == 0u)
            {
                ml[((wave * NT + n) * 16u + r) * 2u] = m[n];
                ml[((wave * NT + n) * 16u + r) * 2u + 1u] = l[n];
            }
        }
    }
};
template <int HD, int NT, uint32_t W>
constexpr uint32_t wave_lds() { return W * (HD / 16u) * NT * 64u * 16u + W * NT * 16u * 2u * 4u; }

// ---- kv4_rows.hip: many query rows, 128 a block, in p.parts parts; what a launch needs
constexpr uint32_t ROWS_BLOCK = 128;
int kv4_rows_launch(opure_dev* dev, const WinParams& p, uint32_t wgs);

// ---- kv4_one.hip: a workgroup has all tiles of a sequence for a block of query rows (p.two: 32, else 16)
uint32_t kv4_one_waves(uint32_t hd, bool two);             // of such a workgroup
int kv4_one_launch(opure_dev* dev, const WinParams& p, uint32_t wgs);

}  // namespace opure_kv4
