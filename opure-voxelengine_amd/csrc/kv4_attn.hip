// ============================================================================
//  kv4_attn.hip -- attention over the 4-bit paged cache (kv4.h), with a sliding
//  window and first positions that stay visible or without.
//
//  Row j of a sequence, at position p = seq_len + j, sees t <= p with t < sinks or
//  t > p - window:  s_t = scale q.k_t,  w_t = exp(s_t - m) / sum exp(s - m),
//  out = sum w_t v_t.
// ============================================================================
#include "kv4.h"
#include "window.h"

#include <algorithm>

using namespace opure_win;
using namespace opure_kv4;
using opure_hip::act_bytes;

namespace {

constexpr uint32_t MAX_PARTS = 64;                         // of a (sequence, KV head, block of query rows): a lane of the joining wave each
constexpr float LOG2E = 1.44269504088896340736f;
// A row's output is scaled to a new maximum only where that passes the old one by 2^LAG.  Weights are held times
// 2^SHIFT, so the largest of 2^15 is still in fp16, and what fp16 loses at its small end lies 2^36 below 1.
constexpr float SHIFT = 12.0f, LAG = 3.0f;

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
                top = fmaxf(top, __builtin_isfinite(x[s][i]) ? __builtin_fabsf(x[s][i]) : 0.0f);
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
// sequence a workgroup 68 us, pieces that end with their sequence 62 to 65.
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

// A workgroup takes a piece of the tiles that the sequences' rows see, for 16 NT query
// rows of a KV head (row qi = j group + head), a wave every fourth tile of 32
// positions of a sequence's part with a running maximum, sum and output of its own in registers.  Lane
// (r, g) holds scores of query row r and the tokens 4 g .. 4 g + 3 of both pages,
// which is its operand P^T in the order that the V codes have.  Each tile's words are
// asked for when the last one's are used up.  The four waves are merged in LDS, the
// parts by k_kv4_join.
//   PIECES: of one size over all sequences, where they are long; else a workgroup has a
// part of one sequence, as many of each.
template <int AF, int HD, int NT, bool ONCE, bool PIECES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NT == 2 ? 2 : HD > 128 ? 1 : AF == OPURE_A_F32 ? 2 : 3))) void k_kv4_split(WinParams p)
{
    typedef Kv4Tile<HD, ONCE> T;
    constexpr uint32_t TT = 32u, DT = HD / 16u, NG = T::NG, QT = AF == OPURE_A_F32 ? 2u : 1u;
    constexpr bool REST = AF != OPURE_A_BF16;              // a weight's rounding rest counts: bf16 results are rounded 2^3 more coarsely than a weight
    extern __shared__ __align__(16) uint8_t lds[];
    f4_t* cacc = reinterpret_cast<f4_t*>(lds);                            // [wave][DT][NT][64]
    float* cml = reinterpret_cast<float*>(lds + 4u * DT * NT * 64u * 16u);   // [wave][NT][16][2]
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t G = p.n_heads / p.n_kv, Gq = G * p.rows;
    // KV heads next to each other, then pieces, or parts, blocks of rows and sequences
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, part = PIECES ? rest : rest % p.parts, group = PIECES ? 0u : rest / p.parts;
    uint32_t b = ONCE ? group : group / p.blocks;
    const uint32_t blk = ONCE ? 0u : group - b * p.blocks, q0 = blk * 16u * NT;
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
    const Bits bits;
    const uint32_t j0 = q0 / G, j1 = min(q0 + 16u * NT - 1u, Gq - 1u) / G;    // the block's first and last row
    const uint32_t page_bytes = p.n_kv * (BLOCK * NG);
    const uint8_t* base = static_cast<const uint8_t*>(p.pool) + block_at(p.layer, p.n_pages, 0u, p.n_kv, kh, NG);
    // ---- the piece's part of sequence b: the wave's tiles i, i + 4, .. below last of its list, its queries and first words
    const int32_t* pt;
    WinSeq sq;
    WinSpan span;
    u4v q[NT][QT][NG];
    uint32_t jr[NT], i, last, has;
    float c[NT];
    int32_t e = -1, pa = -1, pb = -1;
    T tl;
    // pages of tile i of the list: -1 past the sequence, missing or not in the pool
    auto entry = [&](uint32_t i) { return pt[min(span.tile(min(i, span.n - 1u)) * 2u + (lane & 1u), p.max_pages - 1u)]; };
    auto page = [&](int32_t e, uint32_t i, uint32_t which) -> int32_t {
        const int32_t pg = __builtin_amdgcn_readlane(e, which);
        return (span.tile(i) * 2u + which) * OPURE_PAGE_SIZE < sq.total && static_cast<uint32_t>(pg) < p.n_pages ? pg : -1;
    };
    auto at = [&](int32_t pg) { return base + static_cast<uint64_t>(pg < 0 ? 0u : static_cast<uint32_t>(pg)) * page_bytes; };
    auto start = [&]() {
        pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
        sq = win_seq(p, p.seq_len[b]);
        span = seq_span(p, sq);
        has = max(span.n, 1u);
        i = (PIECES ? at0 - before : part_of(p, span.n * part)) + wave;
        last = PIECES ? min(min(at1 - before, has), span.n) : part_of(p, span.n * (part + 1u));
        if (i < last)
        {
            e = entry(i);
            pa = page(e, i, 0u);
            pb = page(e, i, 1u);
            tl.load_k(at(pa), at(pb), lane);
            tl.load_v(at(pa), at(pb), lane);
            e = entry(i + 4u);
        }
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n)
        {
            const uint32_t qi = min(q0 + 16u * n + r, Gq - 1u);
            jr[n] = qi / G;
            c[n] = signed_query<AF, HD, 4>(p, (static_cast<uint64_t>(b) * p.rows + jr[n]) * p.n_heads + kh * G + (qi - jr[n] * G), g, q[n]);
        }
    };
    start();
    while (true)
    {
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
    if (i < last)
        while (true)
        {
            const uint32_t t0 = span.tile(i) * TT;
            const bool more = i + 4u < last;
            const int32_t na = more ? page(e, i + 4u, 0u) : pa, nb = more ? page(e, i + 4u, 1u) : pb;
            if (more) e = entry(i + 8u);
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
                const bool grown = m[n] == NEG_INF ? mx > NEG_INF : __fmul_rn(__fsub_rn(mx, m[n]), c[n]) > LAG;
                if (__any(grown))
                {
                    const float to = grown ? mx : m[n], a = m[n] == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(m[n], to), c[n]));
                    m[n] = to;
                    l[n] = __fmul_rn(l[n], a);
#pragma unroll
                    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
                        for (uint32_t y = 0; y < 4; ++y) o[d][n][y] = __fmul_rn(o[d][n][y], a);
                }
                const float down = m[n] == NEG_INF ? 0.0f : __fsub_rn(SHIFT, __fmul_rn(m[n], c[n]));
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
            i += 4u;
        }
    settle();
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
            cml[((wave * NT + n) * 16u + r) * 2u] = m[n] == NEG_INF ? NEG_INF : __fmul_rn(m[n], c[n]);   // in powers of two
            cml[((wave * NT + n) * 16u + r) * 2u + 1u] = l[n];
        }
    }
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
    __syncthreads();
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
            for (uint32_t y = 0; y < 4; ++y) acc[y] = __fmul_rn(w[0], acc[y]);
#pragma unroll
            for (uint32_t x = 1; x < 4; ++x)
            {
                const f4_t v = cacc[((x * DT + d) * NT + n) * 64u + lane];
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y) acc[y] = __fmaf_rn(w[x], v[y], acc[y]);
            }
            *reinterpret_cast<f4_t*>(p.part_acc + (pbase + qi) * HD + 16u * d + 4u * g) = acc;
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

// ---- many query rows -----------------------------------------------------------

typedef float f16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f16_t mfma_32(u4v a, u4v b, f16_t c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

template <int HD>
constexpr uint32_t rows_pages() { return HD <= 128 ? 4u : 2u; }          // pages a tile
template <int HD>
constexpr uint32_t rows_stage() { return rows_pages<HD>() * (HD / 16u * 512u + groups(HD) * 1024u); }   // bytes of a tile's values in LDS
template <int HD>
constexpr uint32_t rows_lds() { return 2u * rows_stage<HD>(); }
constexpr uint32_t ROWS_BLOCK = 128;

// A workgroup takes 128 query rows (qi = j group + head) of a KV head, 32 a wave, over
// tiles of four pages (two past 128 channels) whose values the waves make from the codes
// once, each its page's, and share in LDS as operands: products are 32x32x16, S^T = K Q^T
// and O^T = V^T P^T.  A lane (q = lane % 32, h = lane / 32) holds of a page's scores the
// tokens 4 h .. 4 h + 3 and 8 + 4 h .. 11 + 4 h of row q, its operand P^T, and V of a
// page lies in LDS in that order of tokens.  Two stages: while one tile is computed the
// next one's words are on their way.
template <int AF, int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD <= 128 ? 2 : 1))) void k_kv4_rows(WinParams p)
{
    constexpr uint32_t NG = groups(HD), KS = HD / 16u, NP = rows_pages<HD>(), TT = 16u * NP, QT = AF == OPURE_A_F32 ? 2u : 1u;
    constexpr bool REST = AF != OPURE_A_BF16, SPLIT = NP == 2u;          // two pages: two waves make K, two V
    extern __shared__ __align__(16) uint8_t lds[];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, h = lane >> 5, r = lane & 31u;
    const uint32_t G = p.n_heads / p.n_kv, Gq = G * p.rows;
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, part = rest % p.parts, b = rest / p.parts / p.blocks;
    const uint32_t blk = p.blocks - 1u - (rest / p.parts - b * p.blocks), q0 = blk * ROWS_BLOCK;    // the rows that see most first
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    const WinSeq sq = win_seq(p, p.seq_len[b]);
    const uint32_t j0 = q0 / G, j1 = min(q0 + ROWS_BLOCK - 1u, Gq - 1u) / G;
    const WinSpan span = win_span<TT>(p, sq, sq.ctx + j0, sq.ctx + j1 + 1u);
    const uint32_t first = span.n * part / p.parts;
    const uint32_t last = span.n * (part + 1u) / p.parts;
    // the wave's rows
    const uint32_t w0 = min(q0 + 32u * wave, Gq - 1u), w1 = min(q0 + 32u * wave + 31u, Gq - 1u), qi = min(w0 + r, Gq - 1u);
    const uint32_t j = qi / G, pos = sq.ctx + j, pos0 = sq.ctx + w0 / G, pos1 = sq.ctx + w1 / G;
    const uint64_t row = (static_cast<uint64_t>(b) * p.rows + j) * p.n_heads + kh * G + (qi - j * G);
    u4v q[QT][KS];
    const float c = signed_query<AF, HD, 2>(p, row, h, q);
    const Bits bits;
    const uint32_t page_bytes = p.n_kv * (BLOCK * NG);
    const uint8_t* base = static_cast<const uint8_t*>(p.pool) + block_at(p.layer, p.n_pages, 0u, p.n_kv, kh, NG);

    // ---- a tile's codes to values: wave w has page w (of two: page w % 2, K or V)
    const uint32_t mine = SPLIT ? wave & 1u : wave;
    const bool has_k = !SPLIT || wave < 2u, has_v = !SPLIT || wave >= 2u;
    uint32_t kw[NG], ks[NG], vw[NG];
    u4v vs[NG];
    int32_t pg = -1, e = -1;                               // the page, and the next one's entry
    auto entry = [&](uint32_t i) { e = pt[min(span.tile(min(i, span.n - 1u)) * NP + mine, p.max_pages - 1u)]; };
    auto fetch = [&](uint32_t i) {
        const uint32_t col = span.tile(i) * NP + mine;
        pg = __builtin_amdgcn_readfirstlane(col * OPURE_PAGE_SIZE < sq.total && static_cast<uint32_t>(e) < p.n_pages ? e : -1);
        const uint8_t* at = base + static_cast<uint64_t>(pg < 0 ? 0u : static_cast<uint32_t>(pg)) * page_bytes;
        if (has_k)
        {
            load_words<NG, false>(reinterpret_cast<const uint32_t*>(at) + lane * NG, kw);
            load_words<NG, false>(reinterpret_cast<const uint32_t*>(at + k_scales(NG)) + (lane & 15u) * NG, ks);
        }
        if (has_v)
        {
            load_words<NG, false>(reinterpret_cast<const uint32_t*>(at + v_codes(NG)) + lane * NG, vw);
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g) vs[g] = win_load<false>(at + v_scales(NG) + ((lane >> 4) * NG + g) * 16u);
        }
    };
    // K of two pages: [step of 16 channels][lane 32 h + 16 (page of two) + token]; V of a page: [32 channels][lane 32 h + channel]
    auto k_at = [&](uint32_t stage, uint32_t pair, uint32_t s) {
        return reinterpret_cast<u4v*>(lds + stage * rows_stage<HD>() + (pair * KS + s) * 1024u);
    };
    auto v_at = [&](uint32_t stage, uint32_t page, uint32_t g) {
        return reinterpret_cast<u4v*>(lds + stage * rows_stage<HD>() + NP * KS * 512u + (page * NG + g) * 1024u);
    };
    auto store = [&](uint32_t i) {
        const uint32_t stage = i & 1u, t0 = span.tile(i) * TT + 16u * mine;
        if (has_k)
        {
            const uint32_t to = (lane >> 4 & 1u) * 32u + (mine & 1u) * 16u + (lane & 15u);
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g)
            {
                // positions without a page: NaN keys for the rows that see them
                const half2_t sb = pair(pg < 0 ? 0x7E007E00u : ks[g]), sc = {sb[0], sb[0]}, ba = {sb[1], sb[1]};
                const u4v k = {values(bits.codes<0>(kw[g]), sc, ba), values(bits.codes<1>(kw[g]), sc, ba), values(bits.codes<2>(kw[g]), sc, ba), values(bits.codes<3>(kw[g]), sc, ba)};
                if (HD % 32 == 0 || g + 1u < NG || lane < 32u) k_at(stage, mine >> 1, 2u * g + (lane >> 5))[to] = k;
            }
        }
        if (has_v)
        {
            const uint32_t x = lane >> 4, t = t0 + 4u * x, n = pg < 0 || t >= sq.total ? 0u : min(sq.total - t, 4u);
            const uint32_t m0 = n >= 2u ? 0xFFFFFFFFu : n == 1u ? 0xFFFFu : 0u, m1 = n >= 4u ? 0xFFFFFFFFu : n == 3u ? 0xFFFFu : 0u;
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g)
            {
                // slots past the sequence and pages that are not there hold anything: 0
                const half2_t s0 = pair(vs[g][0] & m0), s1 = pair(vs[g][1] & m1), b0 = pair(vs[g][2] & m0), b1 = pair(vs[g][3] & m1);
                u2v* to = reinterpret_cast<u2v*>(v_at(stage, mine, g) + (x & 1u) * 32u + (lane & 15u)) + (x >> 1);
                to[0] = u2v{values(bits.codes<0>(vw[g]), s0, b0), values(bits.codes<1>(vw[g]), s1, b1)};
                to[32] = u2v{values(bits.codes<2>(vw[g]), s0, b0), values(bits.codes<3>(vw[g]), s1, b1)};   // 16 channels on
            }
        }
    };

    f16_t o[NG];
    float m = NEG_INF, l = 0.0f;                            // the maximum in units of the products; this lane's share of the sum
#pragma unroll
    for (uint32_t g = 0; g < NG; ++g)
#pragma unroll
        for (uint32_t y = 0; y < 16; ++y) o[g][y] = 0.0f;
    if (first < last)
    {
        entry(first);
        fetch(first);
        entry(first + 1u);
        store(first);
    }
    __syncthreads();
    for (uint32_t i = first; i < last; ++i)
    {
        const uint32_t stage = i & 1u, t0 = span.tile(i) * TT;
        const bool more = i + 1u < last;
        if (more) fetch(i + 1u);
        entry(i + 2u);
        // a tile that none of the wave's rows sees is left out
        const bool none = t0 > pos1 || (t0 >= p.sinks && static_cast<uint64_t>(t0) + TT - 1u + p.window <= pos0);
        if (!none)
        {
            f16_t s[NP / 2u];
#pragma unroll
            for (uint32_t x = 0; x < NP / 2u; ++x)
            {
#pragma unroll
                for (uint32_t y = 0; y < 16; ++y) s[x][y] = 0.0f;
#pragma unroll
                for (uint32_t d = 0; d < KS; ++d)
                {
                    const u4v k = k_at(stage, x, d)[lane];
#pragma unroll
                    for (uint32_t z = 0; z < QT; ++z) s[x] = mfma_32(k, q[z][d], s[x]);
                }
            }
            auto largest = [&]() {
                float v = s[0][0];
#pragma unroll
                for (uint32_t x = 0; x < NP / 2u; ++x)
#pragma unroll
                    for (uint32_t y = 0; y < 16; ++y) v = fmaxf(v, s[x][y]);
                return v;
            };
            float mx = settled(largest());
            // every row of the wave sees every position
            const bool full = t0 + TT <= min(pos0 + 1u, sq.total) && (t0 + TT <= p.sinks || t0 + p.window > pos1);
            if (!full)
            {
                const WinMask mask(p, pos, sq.total, t0 + 4u * h);
#pragma unroll
                for (uint32_t x = 0; x < NP / 2u; ++x)
#pragma unroll
                    for (uint32_t y = 0; y < 16; ++y) s[x][y] = mask.sees(static_cast<int32_t>(32u * x + 8u * (y >> 2) + (y & 3u))) ? s[x][y] : NEG_INF;
                mx = largest();
            }
            mx = max_xor32(mx);
            const bool grown = m == NEG_INF ? mx > NEG_INF : __fmul_rn(__fsub_rn(mx, m), c) > LAG;
            if (__any(grown))
            {
                const float to = grown ? mx : m, a = m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(m, to), c));
                m = to;
                l = __fmul_rn(l, a);
#pragma unroll
                for (uint32_t g = 0; g < NG; ++g)
#pragma unroll
                    for (uint32_t y = 0; y < 16; ++y) o[g][y] = __fmul_rn(o[g][y], a);
            }
            const float down = m == NEG_INF ? 0.0f : __fsub_rn(SHIFT, __fmul_rn(m, c));
#pragma unroll
            for (uint32_t x = 0; x < NP; ++x)
            {
                // a page: 8 scores
                u4v hi, lo;
                float e[8];
#pragma unroll
                for (uint32_t y = 0; y < 8; ++y)
                {
                    e[y] = __builtin_amdgcn_exp2f(__fmaf_rn(s[x >> 1][8u * (x & 1u) + y], c, down));
                    l += e[y];
                }
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y)
                {
                    hi[y] = win_pack<OPURE_A_F16>(e[2 * y], e[2 * y + 1]);
                    if constexpr (REST)
                        lo[y] = win_pack<OPURE_A_F16>(__fsub_rn(e[2 * y], win_low<OPURE_A_F16>(hi[y])), __fsub_rn(e[2 * y + 1], win_high<OPURE_A_F16>(hi[y])));
                }
#pragma unroll
                for (uint32_t g = 0; g < NG; ++g)
                {
                    const u4v v = v_at(stage, x, g)[lane];
                    if constexpr (REST) o[g] = mfma_32(v, lo, o[g]);
                    o[g] = mfma_32(v, hi, o[g]);
                }
            }
        }
        if (more) store(i + 1u);
        __syncthreads();
    }
    settle();
    l = add_xor32(l);
    const bool there = q0 + 32u * wave + r < Gq;
    if (p.parts > 1u)
    {
        const uint64_t at = ((((static_cast<uint64_t>(b) * p.n_kv + kh) * p.blocks + blk) * p.parts + part) * p.block_rows) + 32u * wave + r;
        if (!there) return;
        if (h == 0u)
        {
            // the join takes maxima in powers of two
            p.part_ml[at * 2u] = m == NEG_INF ? NEG_INF : __fmul_rn(m, c);
            p.part_ml[at * 2u + 1u] = l;
        }
#pragma unroll
        for (uint32_t g = 0; g < NG; ++g)
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y)
                if (32u * g + 8u * y < HD)
                    *reinterpret_cast<f4_t*>(p.part_acc + at * HD + 32u * g + 8u * y + 4u * h) = f4_t{o[g][4 * y], o[g][4 * y + 1], o[g][4 * y + 2], o[g][4 * y + 3]};
        return;
    }
    bool fine = true;
    const float by = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    uint8_t* out = static_cast<uint8_t*>(p.out) + row * HD * (AF == OPURE_A_F32 ? 4u : 2u);
#pragma unroll
    for (uint32_t g = 0; g < NG; ++g)
#pragma unroll
        for (uint32_t y = 0; y < 4; ++y)
        {
            if (32u * g + 8u * y >= HD) continue;
            const uint32_t d = 32u * g + 8u * y + 4u * h;
            float v[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
            {
                v[e] = l == 0.0f ? 0.0f : AF == OPURE_A_F32 ? __fdiv_rn(o[g][4 * y + e], l) : __fmul_rn(o[g][4 * y + e], by);
                fine = fine && __builtin_isfinite(v[e]);
            }
            if (!there) continue;
            if constexpr (AF == OPURE_A_F32)
            {
                reinterpret_cast<float2*>(out + d * 4u)[0] = float2{v[0], v[1]};
                reinterpret_cast<float2*>(out + d * 4u)[1] = float2{v[2], v[3]};
            }
            else *reinterpret_cast<u2v*>(out + d * 2u) = u2v{win_pack<AF>(v[0], v[1]), win_pack<AF>(v[2], v[3])};
        }
    // rows that are not finite again, position by position; the loop's last barrier freed the stages
    uint64_t left = __ballot(there && !fine);
    left = (left | left >> 32) & 0xFFFFFFFFu;
    float* const qs = reinterpret_cast<float*>(lds) + wave * 256u;
    while (left)
    {
        const uint32_t x = static_cast<uint32_t>(__builtin_ctzll(left)), qx = w0 + x, jx = qx / G;
        left &= left - 1u;
        const uint64_t at = ((static_cast<uint64_t>(b) * p.rows + jx) * p.n_heads + kh * G + (qx - jx * G)) * HD;
        __builtin_amdgcn_wave_barrier();
        for (uint32_t d = lane; d < HD; d += 64u) qs[d] = load_act<AF>(p.q, at + d);
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float lx, v[4];
        kv4_row(p, qs, b, kh, sq.ctx + jx, sq.total, lx, v);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (lane + 64u * e < HD) store_act_rt(p.out, at + lane + 64u * e, lx == 0.0f ? 0.0f : __fdiv_rn(v[e], lx), AF);
    }
}

template <int HD, int NT>
constexpr uint32_t split_lds() { return 4u * (HD / 16u) * NT * 64u * 16u + 4u * NT * 16u * 2u * 4u; }

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
        const int rc = win_lds(dev, reinterpret_cast<const void*>(kernel), split_lds<HD, NT>(), done);
        if (rc) return rc;
        int n = a_cu.load(std::memory_order_relaxed);
        if (n == 0)
        {
            OPURE_HIP_TRY(hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, split_lds<HD, NT>()));
            n = std::max(n, 1);
            a_cu.store(n, std::memory_order_relaxed);
        }
        return f(kernel, split_lds<HD, NT>(), static_cast<uint32_t>(n) * (dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u));
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

// The same of the kernel of many query rows.
template <typename F>
int rows_kernel(opure_dev* dev, uint32_t afmt, uint32_t hd, F&& f)
{
    auto by_head = [&](auto af) {
        return win_by_head(hd, [&](auto h) {
            constexpr int AF = decltype(af)::value, HD = decltype(h)::value;
            static std::atomic<uint64_t> done{0};
            auto* kernel = &k_kv4_rows<AF, HD>;
            const int rc = win_lds(dev, reinterpret_cast<const void*>(kernel), rows_lds<HD>(), done);
            return rc ? rc : f(kernel, rows_lds<HD>());
        });
    };
    return afmt == OPURE_A_F32   ? by_head(std::integral_constant<int, OPURE_A_F32>{})
           : afmt == OPURE_A_F16 ? by_head(std::integral_constant<int, OPURE_A_F16>{})
                                 : by_head(std::integral_constant<int, OPURE_A_BF16>{});
}

// How a call is split, and its workspace.
struct Kv4Plan {
    uint32_t tiles = 0, blocks = 0, block_rows = 0, parts = 0, least = 1;
    bool two = false, many = false, pieces = false;      // blocks of 32 query rows, of 128; pieces of one size
    uint64_t acc = 0, ml = 0;                            // bytes
    uint64_t bytes() const { return acc + ml; }
};

// workspace of `slots` parts' outputs, and what a launch can have
int kv4_slots(const opure_attn_kv4_args* a, uint64_t slots, uint64_t wgs, uint64_t rows, Kv4Plan& w)
{
    w.acc = opure_hip::align_up(slots * w.block_rows * a->model->head_dim * 4u, 256);
    w.ml = opure_hip::align_up(slots * w.block_rows * 8u, 256);
    // a launch's threads, 256 a workgroup (the join's: a row at most), stay in 32 bits
    OPURE_REQUIRE(std::max(wgs, rows) < 1u << 24, OPURE_E_CAPACITY, "4-bit attention: %u x %u rows of %u heads over max_ctx %u: too many workgroups",
                  a->batch, a->rows, a->model->n_heads, a->max_ctx);
    return OPURE_OK;
}

int kv4_plan(opure_dev* dev, const opure_attn_kv4_args* a, Kv4Plan& w)
{
    const opure_model* m = a->model;
    const uint32_t Gq = m->n_heads / m->n_kv_heads * a->rows;
    // tiles of any block of rows: its sinks', then the window's and the rows', which begin anywhere in a tile
    const uint64_t all = (a->max_ctx + 31u) / 32u, window = a->window ? a->window : 0x7FFFFFFFu;
    w.tiles = static_cast<uint32_t>(std::min<uint64_t>(all, (a->sinks + 31ull) / 32u + (window + a->rows + 30ull) / 32u + 1u));
    const uint64_t heads = static_cast<uint64_t>(a->batch) * m->n_kv_heads, rows = heads * Gq;
    const uint64_t cu = dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u;
    w.many = Gq > 64u;
    if (w.many)
    {
        w.blocks = (Gq + ROWS_BLOCK - 1u) / ROWS_BLOCK;
        w.block_rows = std::min(Gq, ROWS_BLOCK);
        w.parts = static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>(1u, 2u * cu / (heads * w.blocks)), std::min((w.tiles + 7u) / 8u, MAX_PARTS)));
        const uint64_t wgs = heads * w.blocks * w.parts;
        return kv4_slots(a, w.parts == 1u ? 0u : wgs, wgs, rows, w);
    }
    w.two = Gq > 16u && m->head_dim <= 128u;
    w.blocks = (Gq + (w.two ? 31u : 15u)) / (w.two ? 32u : 16u);
    w.block_rows = std::min(Gq, w.two ? 32u : 16u);
    uint32_t room = 0;
    auto holds = [&](auto, uint32_t, uint32_t n) {
        room = n;
        return OPURE_OK;
    };
    const uint64_t groups = heads * w.blocks;
    if (w.blocks == 1u && a->batch > 1u)
    {
        int rc = split_kernel(dev, m->afmt, m->head_dim, w.two, true, true, holds);
        if (rc) return rc;
        const uint64_t hold = std::max<uint64_t>(1u, room / m->n_kv_heads), all = static_cast<uint64_t>(a->batch) * w.tiles;
        w.pieces = !w.two && all >= 32u * hold;
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
    rc = w.many ? rows_kernel(dev, p.afmt, p.hd, launch) : split_kernel(dev, p.afmt, p.hd, w.two, w.blocks == 1u, w.pieces, launch);
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
