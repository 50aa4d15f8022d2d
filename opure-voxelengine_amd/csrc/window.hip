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
#include "internal.h"

#include <algorithm>
#include <atomic>

using namespace opure_dev_math;

namespace {

struct WinParams {
    const void* q;
    void* out;
    const void* pool;
    const int32_t* page_table;
    const int32_t* seq_len;
    float* part_acc;     // [batch][n_kv][parts][Gq][hd]: a part's unnormalised output of each query row
    float* part_ml;      // [batch][n_kv][parts][Gq][2]: its maximum (in powers of two) and sum
    float* scores;       // with weights: [batch][n_kv][tiles][Gq][tile's positions], in powers of two
    float* weights;
    uint64_t weights_batch_stride;
    uint32_t weights_stride;
    uint32_t n_heads, n_kv, hd, rows, n_pages, max_pages, layer, afmt;
    uint32_t window, sinks;       // window >= 1: 2^31 - 1 sees everything
    uint32_t cap;                 // positions that may be read: min(max_ctx, the table's)
    uint32_t parts, blocks;       // parts a (sequence, KV head, block of query rows); such blocks
    uint32_t tiles;               // most tiles a sequence's rows see
    uint32_t combine_rows;        // query rows of the call
    uint32_t combine_wgs;         // k_win_join: its first workgroups join the parts, the others add the weights
    float scale;
    uint32_t* err;
};

// A sequence's positions: `ctx` before the rows, `total` that may be read.  A
// negative length or one that passes the capacity is reported and clamped.
struct WinSeq {
    uint32_t ctx, total;
};

__device__ __forceinline__ WinSeq win_seq(const WinParams& p, int32_t len)
{
    WinSeq s;
    s.ctx = len < 0 ? 0u : static_cast<uint32_t>(len);
    s.total = min(s.ctx + p.rows, p.cap);
    if ((len < 0 || s.ctx + p.rows > p.cap) && threadIdx.x == 0u && p.err) p.err[ERR_POSITION] = 1u;
    return s;
}

__device__ __forceinline__ bool win_sees(const WinParams& p, uint32_t pos, uint32_t t)
{
    return t <= pos && (t < p.sinks || t + p.window > pos);
}

// the page of position t (t < total), or -1
__device__ __forceinline__ int32_t win_page(const WinParams& p, const int32_t* pt, uint32_t t)
{
    const int32_t pg = pt[t / OPURE_PAGE_SIZE];
    return pg >= 0 && static_cast<uint32_t>(pg) < p.n_pages ? pg : -1;
}

// One query row by one wave, exactly as the formulas say it: lanes over 64
// positions for the scores, then over channels for the output; a position that
// the row does not see is not read.  qs: the row in LDS (hd floats).
__device__ void win_row(const WinParams& p, const float* qs, uint32_t b, uint32_t kh, uint32_t pos, uint32_t total,
                        float& m, float& l, float (&o)[4])
{
    const uint32_t lane = threadIdx.x & 63u, hd = p.hd;
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    const uint32_t end = min(pos + 1u, total);
    const uint32_t low = pos + 1u > p.window ? pos + 1u - p.window : 0u;   // the window's first position
    m = -__builtin_huge_valf();
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
        float s = -__builtin_huge_valf();
        if (in && pg < 0) s = __builtin_nanf("");
        if (in && pg >= 0)
        {
            const uint64_t at = kv_elem(p.layer, p.n_pages, static_cast<uint32_t>(pg), 0u, p.n_kv, kh, hd, t % OPURE_PAGE_SIZE, 0u);
            float acc = 0.0f;
            for (uint32_t d = 0; d < hd; ++d) acc = __fmaf_rn(qs[d], load_act_rt(p.pool, at + d, p.afmt), acc);
            s = __fmul_rn(acc, p.scale);
        }
        const float mx = fmaxf(m, wave_max64(s));          // a NaN score leaves the maximum and reaches the sum
        const float ms = mx == -__builtin_huge_valf() ? 0.0f : mx;
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
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const uint32_t d = lane + 64u * i;
                if (d < hd)
                    o[i] = __fmaf_rn(w, load_act_rt(p.pool, kv_elem(p.layer, p.n_pages, pk, 1u, p.n_kv, kh, hd, tk % OPURE_PAGE_SIZE, d),
                                                    p.afmt), o[i]);
            }
        }
    }
}

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr float NEG_INF = -__builtin_huge_valf();

// The tiles (TT positions each) that the rows at ctx .. ctx + rows - 1 see: the
// sinks' first, then the window's.  Tile i of the list starts at position start(i).
struct WinSpan {
    uint32_t ns, w0, n;           // sink tiles, the window's first tile, tiles in all
    __device__ __forceinline__ uint32_t tile(uint32_t i) const { return i < ns ? i : i - ns + w0; }
};

template <uint32_t TT>
__device__ __forceinline__ WinSpan win_span(const WinParams& p, const WinSeq& sq, uint32_t first_pos, uint32_t end_pos)
{
    WinSpan s;
    const uint32_t low = first_pos + 1u > p.window ? first_pos + 1u - p.window : 0u;
    const uint32_t end = min(end_pos, sq.total);
    const uint32_t last = (end + TT - 1u) / TT;
    s.w0 = min(low / TT, last);
    s.ns = min((min(p.sinks, end) + TT - 1u) / TT, s.w0);
    s.n = s.ns + last - s.w0;
    return s;
}

// Operands of S^T = K Q^T and O^T = V^T P^T by 16x16 matrix instructions, lane
// (r = lane % 16, g = lane / 16).  A tile is 32 positions of a 16-bit cache, two
// score blocks of 16: row r of block T is position 8 (r / 4) + r % 4 + 4 T, so
// that a lane's scores are positions 8 g .. 8 g + 7, which is its operand P^T,
// and its part of a V channel is 16 bytes.  In fp32 a tile is one page, row r is
// position r, a lane's scores are positions 4 g .. 4 g + 3 and each of the four
// takes a matrix instruction over 4 positions.
template <int AF, int HD>
struct WinTile {
    static constexpr uint32_t EB = AF == OPURE_A_F32 ? 4u : 2u, TT = AF == OPURE_A_F32 ? 16u : 32u, NB = TT / 16u;
    static constexpr uint32_t KS = AF == OPURE_A_F32 ? HD / 16u : (HD + 31u) / 32u, DT = HD / 16u, NS = 16u / EB;
    static constexpr uint32_t PB = OPURE_PAGE_SIZE * HD * EB;   // bytes of a K or V plane
    static constexpr bool HALF = AF != OPURE_A_F32 && HD % 32 != 0;   // the last step's upper channels are not there
    u4v k[NB][KS], v[DT];

    __device__ __forceinline__ static float part(u4v x, uint32_t i) { return __uint_as_float(x[i]); }
    __device__ __forceinline__ void load_k(const uint8_t* a, const uint8_t* b, uint32_t r, uint32_t g)
    {
        const uint8_t* at = AF == OPURE_A_F32 || r < 8u ? a : b;
        const uint32_t slot = AF == OPURE_A_F32 ? r : 8u * ((r >> 2) & 1u) + (r & 3u);
        at += slot * (HD * EB) + 16u * g;
#pragma unroll
        for (uint32_t t = 0; t < NB; ++t)
#pragma unroll
            for (uint32_t s = 0; s < KS; ++s)
            {
                if (HALF && s + 1u == KS && g >= 2u) k[t][s] = u4v{0u, 0u, 0u, 0u};
                else k[t][s] = *reinterpret_cast<const u4v*>(at + t * 4u * HD * EB + 64u * s);
            }
    }
    __device__ __forceinline__ void load_v(const uint8_t* a, const uint8_t* b, uint32_t r, uint32_t g)
    {
        const uint8_t* at = AF == OPURE_A_F32 || g < 2u ? a : b;
        at += r * (16u * EB) + (AF == OPURE_A_F32 ? g : (g & 1u)) * 16u;
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d) v[d] = *reinterpret_cast<const u4v*>(at + d * 16u * 16u * EB);
    }
};

template <int AF, int HD>
__device__ __forceinline__ void win_load_q(const WinParams& p, uint64_t row, uint32_t g, u4v (&q)[WinTile<AF, HD>::KS])
{
    typedef WinTile<AF, HD> T;
    const uint8_t* at = static_cast<const uint8_t*>(p.q) + row * (HD * T::EB) + 16u * g;
#pragma unroll
    for (uint32_t s = 0; s < T::KS; ++s)
    {
        if (T::HALF && s + 1u == T::KS && g >= 2u) q[s] = u4v{0u, 0u, 0u, 0u};
        else q[s] = *reinterpret_cast<const u4v*>(at + 64u * s);
    }
}

template <int AF>
__device__ __forceinline__ f4_t win_mfma(u4v a, u4v b, f4_t c)
{
    if constexpr (AF == OPURE_A_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else if constexpr (AF == OPURE_A_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
    {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    }
}

template <int AF>
__device__ __forceinline__ uint32_t win_pack(float a, float b)
{
    typedef float f2v __attribute__((ext_vector_type(2)));
    typedef _Float16 h2v __attribute__((ext_vector_type(2)));
    typedef __bf16 b2v __attribute__((ext_vector_type(2)));
    const f2v v = {a, b};
    if constexpr (AF == OPURE_A_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2v));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2v));
}

template <int AF>
__device__ __forceinline__ float win_low(uint32_t v) { return AF == OPURE_A_F16 ? f16_to_f32(static_cast<uint16_t>(v)) : bits_f(v << 16); }
template <int AF>
__device__ __forceinline__ float win_high(uint32_t v) { return AF == OPURE_A_F16 ? f16_to_f32(static_cast<uint16_t>(v >> 16)) : bits_f(v & 0xFFFF0000u); }

// elements n .. of a 16-byte piece of consecutive positions read 0
template <int AF>
__device__ __forceinline__ u4v win_tail(u4v v, uint32_t n)
{
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
    {
        if (AF == OPURE_A_F32) v[i] = i < n ? v[i] : 0u;
        else v[i] = 2u * i + 1u < n ? v[i] : 2u * i < n ? v[i] & 0xFFFFu : 0u;
    }
    return v;
}

// One tile's scores of a block of query rows, in powers of two (scale log2 e q.k),
// -inf where the row at `pos` does not see the position.
template <int AF, int HD>
__device__ __forceinline__ void win_scores(const WinParams& p, const WinTile<AF, HD>& tl, const u4v (&q)[WinTile<AF, HD>::KS], float c,
                                           bool full, uint32_t t0, uint32_t g, uint32_t pos, uint32_t total,
                                           float (&s)[WinTile<AF, HD>::NS])
{
    typedef WinTile<AF, HD> T;
#pragma unroll
    for (uint32_t t = 0; t < T::NB; ++t)
    {
        f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t k = 0; k < T::KS; ++k) acc = win_mfma<AF>(tl.k[t][k], q[k], acc);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) s[4u * t + i] = __fmul_rn(acc[i], c);
    }
    if (!full)
    {
#pragma unroll
        for (uint32_t i = 0; i < T::NS; ++i)
        {
            const uint32_t t = t0 + T::NS * g + i;
            s[i] = t < total && win_sees(p, pos, t) ? s[i] : NEG_INF;
        }
    }
}

// Few query rows: a workgroup takes a part of the tiles that a sequence's rows
// see, for 16 NT query rows of a KV head (row qi = j group + head), a wave every
// fourth tile with a running maximum, sum and output of its own in registers.
// Bound by the cache's bytes.  A tile's K goes to the matrix unit and the next
// one's loads into the same registers at once, its V likewise, so a wave has
// about a tile (16 KB at 128 channels) in flight all the time without a second
// set of registers.  The four waves are merged in LDS, the parts by k_win_join.
//   A probability enters its product as two 16-bit numbers (its rounding and the
// rest: 16 bits of bf16, 22 of fp16): the products are not what bounds this.
template <int AF, int HD, int NT>
__global__ __launch_bounds__(256) void k_win_split(WinParams p)
{
    typedef WinTile<AF, HD> T;
    constexpr uint32_t TT = T::TT, DT = T::DT, NS = T::NS;
    extern __shared__ __align__(16) uint8_t lds[];
    f4_t* cacc = reinterpret_cast<f4_t*>(lds);                            // [wave][DT][NT][64]
    float* cml = reinterpret_cast<float*>(lds + 4u * DT * NT * 64u * 16u);   // [wave][NT][16][2]
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, part = rest % p.parts;
    const uint32_t b = rest / p.parts / p.blocks, blk = rest / p.parts - b * p.blocks;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t G = p.n_heads / p.n_kv, Gq = G * p.rows, q0 = blk * 16u * NT;
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
        tl.load_k(at(pa), at(pb), r, g);
        tl.load_v(at(pa) + vofs, at(pb) + vofs, r, g);
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
            if (more) tl.load_k(at(na), at(nb), r, g);
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
            tl.load_v(at(na) + vofs, at(nb) + vofs, r, g);
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
    const uint64_t pbase = ((static_cast<uint64_t>(b) * p.n_kv + kh) * p.parts + part) * Gq;
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
    {
        const uint32_t qi = q0 + 16u * n + r;
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
        if (qi >= Gq) continue;
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

// A row's result from its parts' maxima and sums: lane x holds part x's weight.
__device__ __forceinline__ void win_join(const WinParams& p, uint64_t pbase, uint32_t Gq, uint32_t qi, uint32_t lane, float& M, float& w, float& L)
{
    const uint64_t at = (pbase + static_cast<uint64_t>(min(lane, p.parts - 1u)) * Gq + qi) * 2u;
    const float m = p.part_ml[at], l = p.part_ml[at + 1u];
    M = wave_max64(m);
    w = lane < p.parts ? __builtin_amdgcn_exp2f(__fsub_rn(m, M == NEG_INF ? 0.0f : M)) : 0.0f;
    L = wave_sum64(__fmul_rn(w, l));
}

// Joins the parts, a wave a query row: lanes over the parts for the weights, over
// channels for the output.  A row that is not finite is computed again position
// by position: a NaN or an infinity among the values of a position that the row
// does not see meets weight 0 in the products above.  With weights, the launch's
// other workgroups add them: a thread a position, over the query rows in order.
template <uint32_t TT>
__global__ __launch_bounds__(256) void k_win_join(WinParams p)
{
    __shared__ float sm[4][256];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u, G = p.n_heads / p.n_kv, Gq = G * p.rows;
    if (blockIdx.x < p.combine_wgs)
    {
        const uint64_t id = 4ull * blockIdx.x + wave;
        if (id >= p.combine_rows) return;
        const uint32_t head = static_cast<uint32_t>(id % p.n_heads), row = static_cast<uint32_t>(id / p.n_heads), b = row / p.rows, j = row - b * p.rows;
        const uint32_t kh = head / G, qi = j * G + (head - kh * G);
        const uint64_t pbase = (static_cast<uint64_t>(b) * p.n_kv + kh) * p.parts * Gq;
        float M, w, L, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        win_join(p, pbase, Gq, qi, lane, M, w, L);
        for (uint32_t x = 0; x < p.parts; ++x)
        {
            const float wx = __shfl(w, x);
            const float* acc = p.part_acc + (pbase + static_cast<uint64_t>(x) * Gq + qi) * p.hd;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (lane + 64u * i < p.hd) o[i] = __fmaf_rn(wx, acc[lane + 64u * i], o[i]);
        }
        bool fine = true;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
        {
            o[i] = L == 0.0f ? 0.0f : __fdiv_rn(o[i], L);
            fine = fine && __builtin_isfinite(o[i]);
        }
        const uint64_t at = (static_cast<uint64_t>(row) * p.n_heads + head) * p.hd;
        if (!__all(fine))
        {
            for (uint32_t d = lane; d < p.hd; d += 64u) sm[wave][d] = load_act_rt(p.q, at + d, p.afmt);
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const WinSeq sq = win_seq(p, p.seq_len[b]);
            float m, l;
            win_row(p, sm[wave], b, kh, sq.ctx + j, sq.total, m, l, o);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) o[i] = l == 0.0f ? 0.0f : __fdiv_rn(o[i], l);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (lane + 64u * i < p.hd) store_act_rt(p.out, at + lane + 64u * i, o[i], p.afmt);
        return;
    }
    // ---- weights: 256 positions of a (sequence, KV head)
    const uint32_t per = (p.tiles * TT + 255u) / 256u, id = blockIdx.x - p.combine_wgs;
    const uint32_t x = id % per, bh = id / per, kh = bh % p.n_kv, b = bh / p.n_kv;
    const WinSeq sq = win_seq(p, p.seq_len[b]);
    const WinSpan span = win_span<TT>(p, sq, sq.ctx, sq.ctx + p.rows);
    if (x * 256u >= span.n * TT) return;                      // whole workgroup
    const uint32_t at = x * 256u + threadIdx.x, i = at / TT, off = at - i * TT;
    const uint32_t t = i < span.n ? span.tile(i) * TT + off : sq.total;
    const bool in = t < sq.total;
    const uint64_t pbase = static_cast<uint64_t>(bh) * p.parts * Gq;
    const float* s = p.scores + ((static_cast<uint64_t>(bh) * p.tiles + (in ? i : 0u)) * Gq) * TT + off;
    float sum = 0.0f;
    bool any = false;
    for (uint32_t c0 = 0; c0 < Gq; c0 += 128u)
    {
        const uint32_t n = min(128u, Gq - c0);
        __syncthreads();
        for (uint32_t y = wave; y < n; y += 4u)
        {
            float M, w, L;
            win_join(p, pbase, Gq, c0 + y, lane, M, w, L);
            if (lane == 0u)
            {
                sm[0][y] = M == NEG_INF ? 0.0f : M;
                sm[1][y] = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
            }
        }
        __syncthreads();
        if (in)
            for (uint32_t y = 0; y < n; ++y)
            {
                const float v = s[static_cast<uint64_t>(c0 + y) * TT];
                const bool sees = win_sees(p, sq.ctx + (c0 + y) / G, t);
                any = any || sees;
                sum += sees ? __fmul_rn(__builtin_amdgcn_exp2f(__fsub_rn(v, sm[0][y])), sm[1][y]) : 0.0f;
            }
    }
    if (in && any) p.weights[b * p.weights_batch_stride + static_cast<uint64_t>(kh) * p.weights_stride + t] += sum;
}

template <int AF, int HD, int NT>
int win_split_launch(opure_dev* dev, const WinParams& p, uint32_t batch)
{
    constexpr uint32_t lds = 4u * (HD / 16u) * NT * 64u * 16u + 4u * NT * 16u * 2u * 4u;
    if constexpr (lds > 64u * 1024u)
    {
        static std::atomic<uint64_t> done{0};              // a bit a device
        const uint64_t bit = 1ull << (dev->ordinal & 63);
        if (!(done.load(std::memory_order_relaxed) & bit))
            OPURE_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_win_split<AF, HD, NT>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    OPURE_LAUNCH(dev, (k_win_split<AF, HD, NT>), dim3(p.n_kv * p.parts * batch * p.blocks), dim3(256), lds, p);
    OPURE_LAUNCH_CHECK("k_win_split");
    return OPURE_OK;
}

template <int AF, int HD>
int win_split_hd(opure_dev* dev, const WinParams& p, uint32_t batch, bool two)
{
    if constexpr (HD <= 128)
        if (two) return win_split_launch<AF, HD, 2>(dev, p, batch);
    return win_split_launch<AF, HD, 1>(dev, p, batch);
}

template <int AF>
int win_split_any(opure_dev* dev, const WinParams& p, uint32_t batch, bool two)
{
    switch (p.hd / 16u)
    {
    case 1: return win_split_hd<AF, 16>(dev, p, batch, two);
    case 2: return win_split_hd<AF, 32>(dev, p, batch, two);
    case 3: return win_split_hd<AF, 48>(dev, p, batch, two);
    case 4: return win_split_hd<AF, 64>(dev, p, batch, two);
    case 5: return win_split_hd<AF, 80>(dev, p, batch, two);
    case 6: return win_split_hd<AF, 96>(dev, p, batch, two);
    case 7: return win_split_hd<AF, 112>(dev, p, batch, two);
    case 8: return win_split_hd<AF, 128>(dev, p, batch, two);
    case 9: return win_split_hd<AF, 144>(dev, p, batch, two);
    case 10: return win_split_hd<AF, 160>(dev, p, batch, two);
    case 11: return win_split_hd<AF, 176>(dev, p, batch, two);
    case 12: return win_split_hd<AF, 192>(dev, p, batch, two);
    case 13: return win_split_hd<AF, 208>(dev, p, batch, two);
    case 14: return win_split_hd<AF, 224>(dev, p, batch, two);
    case 15: return win_split_hd<AF, 240>(dev, p, batch, two);
    default: return win_split_hd<AF, 256>(dev, p, batch, two);
    }
}

// How a call is split, and its workspace.
struct WinPlan {
    uint32_t tt, tiles, blocks, parts;
    bool two;
    uint64_t acc, ml, scores;     // bytes
    uint64_t bytes() const { return acc + ml + scores; }
};

WinPlan win_plan(const opure_dev* dev, const opure_attn_window_args* a)
{
    const opure_model* m = a->model;
    const uint32_t Gq = m->n_heads / m->n_kv_heads * a->rows, n_cu = dev->n_cu > 0 ? static_cast<uint32_t>(dev->n_cu) : 256u;
    WinPlan w{};
    w.tt = m->afmt == OPURE_A_F32 ? 16u : 32u;
    // tiles of any sequence of the call: its sinks', then the window's and the rows', which begin anywhere in a tile
    const uint64_t all = (a->max_ctx + w.tt - 1u) / w.tt, window = a->window ? a->window : 0x7FFFFFFFu;
    w.tiles = static_cast<uint32_t>(std::min<uint64_t>(all, (a->sinks + w.tt - 1ull) / w.tt + (window + a->rows + w.tt - 2ull) / w.tt + 1u));
    w.two = Gq > 16u && m->head_dim <= 128u;
    w.blocks = (Gq + (w.two ? 31u : 15u)) / (w.two ? 32u : 16u);
    const uint64_t groups = static_cast<uint64_t>(a->batch) * m->n_kv_heads * w.blocks;
    const uint64_t want = (4ull * n_cu + groups - 1u) / groups;
    w.parts = static_cast<uint32_t>(std::min<uint64_t>(want, std::min((w.tiles + 3u) / 4u, 64u)));
    const uint64_t rows = static_cast<uint64_t>(a->batch) * m->n_kv_heads * Gq;
    w.acc = opure_hip::align_up(rows * w.parts * m->head_dim * 4u, 256);
    w.ml = opure_hip::align_up(rows * w.parts * 8u, 256);
    w.scores = a->weights ? opure_hip::align_up(rows * w.tiles * w.tt * 4u, 256) : 0u;
    return w;
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
    // the launches' workgroups and the query rows' indexes stay in 32 bits
    OPURE_REQUIRE(static_cast<uint64_t>(m->n_heads) * a->batch * a->rows <= 1u << 25 && static_cast<uint64_t>(m->n_kv_heads) * a->batch * (a->max_ctx / 64u + 1ull) <= 1u << 24,
                  OPURE_E_CAPACITY, "window attention: %u x %u rows of %u heads, max_ctx %u", a->batch, a->rows, m->n_heads, a->max_ctx);
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
    return ensure_workspace(dev, win_plan(dev, a).bytes());
}

extern "C" int opure_attn_window_paged(opure_dev* dev, const opure_attn_window_args* a)
{
    OPURE_REQUIRE(dev && a && a->q && a->out && a->seq_len, OPURE_E_INVALID, "opure_attn_window_paged: null argument");
    int rc = win_validate(a);
    if (rc) return rc;
    OPURE_REQUIRE((reinterpret_cast<uintptr_t>(a->q) & 15u) == 0u && (reinterpret_cast<uintptr_t>(a->out) & 7u) == 0u &&
                      ((reinterpret_cast<uintptr_t>(a->seq_len) | reinterpret_cast<uintptr_t>(a->weights)) & 3u) == 0u,
                  OPURE_E_INVALID, "opure_attn_window_paged: q must be 16-byte aligned, out 8-byte, seq_len and weights 4-byte");
    const DeviceGuard on(dev);
    const WinPlan w = win_plan(dev, a);
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
    p.scores = a->weights ? p.part_ml + w.ml / 4u : nullptr;
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
    p.tiles = w.tiles;
    p.combine_rows = a->batch * a->rows * p.n_heads;
    p.combine_wgs = (p.combine_rows + 3u) / 4u;
    rc = p.afmt == OPURE_A_F32   ? win_split_any<OPURE_A_F32>(dev, p, a->batch, w.two)
         : p.afmt == OPURE_A_F16 ? win_split_any<OPURE_A_F16>(dev, p, a->batch, w.two)
                                 : win_split_any<OPURE_A_BF16>(dev, p, a->batch, w.two);
    if (rc) return rc;
    const uint32_t sums = p.weights ? (w.tiles * w.tt + 255u) / 256u * p.n_kv * a->batch : 0u;
    if (w.tt == 16u) OPURE_LAUNCH(dev, (k_win_join<16u>), dim3(p.combine_wgs + sums), dim3(256), 0, p);
    else OPURE_LAUNCH(dev, (k_win_join<32u>), dim3(p.combine_wgs + sums), dim3(256), 0, p);
    OPURE_LAUNCH_CHECK("k_win_join");
    return OPURE_OK;
}
