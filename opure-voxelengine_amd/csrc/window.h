// ============================================================================
//  window.h -- what the kernels of windowed attention share: the call's
//  parameters, which positions a row sees, tiles of the paged cache as operands
//  of the matrix instructions, and a query row computed position by position.
// ============================================================================
#pragma once
#include "internal.h"

#include <atomic>
#include <type_traits>

namespace opure_win {

using namespace opure_dev_math;

struct WinParams {
    const void* q;
    void* out;
    const void* pool;
    const int32_t* page_table;
    const int32_t* seq_len;
    float* part_acc;     // [slot][block_rows][hd]: a part's unnormalised output of its block's query rows
    float* part_ml;      // [slot][block_rows][2]: their maxima (in powers of two) and sums
    float* scores;       // with weights: [batch][n_kv][tiles][Gq][tile's positions], in powers of two
    float* lse;          // with weights summed by k_win_sums: [batch][n_kv][Gq], log2 of each row's sum of 2^score
    float* weights;
    uint64_t weights_batch_stride;
    uint32_t weights_stride;
    uint32_t n_heads, n_kv, hd, rows, n_pages, max_pages, layer, afmt;
    uint32_t window, sinks;       // window >= 1: 2^31 - 1 sees everything
    uint32_t cap;                 // positions that may be read: min(max_ctx, the table's)
    uint32_t batch;               // k_win_sums: sequences
    uint32_t sum_rows;            // k_win_sums: query rows a chunk
    uint32_t blocks, block_rows;  // blocks of query rows a (sequence, KV head), and the most rows in one
    uint32_t two;                 // blocks of 32 query rows, not 16
    uint32_t parts;               // parts of each (sequence, KV head, block): slot part + parts * its index
    uint32_t tiles;               // most tiles a sequence's rows see
    uint32_t pieces, least, by_parts;   // 4-bit attention: parts are pieces of one size, its least; 2^32 / parts, rounded up
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
__device__ inline void win_row(const WinParams& p, const float* qs, uint32_t b, uint32_t kh, uint32_t pos, uint32_t total,
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

// a 16-byte load; ONCE: of bytes that no other workgroup reads, kept out of the way of those in the caches
template <bool ONCE>
__device__ __forceinline__ u4v win_load(const uint8_t* p)
{
    const u4v* q = reinterpret_cast<const u4v*>(p);
    if constexpr (ONCE) return __builtin_nontemporal_load(q);
    else return *q;
}

constexpr float NEG_INF = -__builtin_huge_valf();

// The tiles (TT positions each) that the rows at ctx .. ctx + rows - 1 see: the
// sinks' first, then the window's.  Tile i of the list starts at position TT tile(i).
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

    template <bool ONCE>
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
                else k[t][s] = win_load<ONCE>(at + t * 4u * HD * EB + 64u * s);
            }
    }
    template <bool ONCE>
    __device__ __forceinline__ void load_v(const uint8_t* a, const uint8_t* b, uint32_t r, uint32_t g)
    {
        const uint8_t* at = AF == OPURE_A_F32 || g < 2u ? a : b;
        at += r * (16u * EB) + (AF == OPURE_A_F32 ? g : (g & 1u)) * 16u;
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d) v[d] = win_load<ONCE>(at + d * 16u * 16u * EB);
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

// a head size's kernel: f(std::integral_constant<int, HD>)
template <typename F>
int win_by_head(uint32_t hd, F&& f)
{
    switch (hd / 16u)
    {
    case 1: return f(std::integral_constant<int, 16>{});
    case 2: return f(std::integral_constant<int, 32>{});
    case 3: return f(std::integral_constant<int, 48>{});
    case 4: return f(std::integral_constant<int, 64>{});
    case 5: return f(std::integral_constant<int, 80>{});
    case 6: return f(std::integral_constant<int, 96>{});
    case 7: return f(std::integral_constant<int, 112>{});
    case 8: return f(std::integral_constant<int, 128>{});
    case 9: return f(std::integral_constant<int, 144>{});
    case 10: return f(std::integral_constant<int, 160>{});
    case 11: return f(std::integral_constant<int, 176>{});
    case 12: return f(std::integral_constant<int, 192>{});
    case 13: return f(std::integral_constant<int, 208>{});
    case 14: return f(std::integral_constant<int, 224>{});
    case 15: return f(std::integral_constant<int, 240>{});
    default: return f(std::integral_constant<int, 256>{});
    }
}

// Dynamic LDS past 64 KB is asked for once a kernel and device: `done` has a bit a device.
inline int win_lds(const opure_dev* dev, const void* kernel, uint32_t bytes, std::atomic<uint64_t>& done)
{
    const uint64_t bit = 1ull << (dev->ordinal & 63);
    if (bytes <= 64u * 1024u || done.load(std::memory_order_relaxed) & bit) return OPURE_OK;
    OPURE_HIP_TRY(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    done.fetch_or(bit, std::memory_order_relaxed);
    return OPURE_OK;
}

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

// What a row sees of the positions from `base` on, base + y being visible where
// y <= end and (y < sinks or y >= low): y is a constant, so a mask is three
// comparisons with one, and nothing of it has to be kept across a loop.
struct WinMask {
    int32_t end, sinks, low;
    __device__ __forceinline__ WinMask(const WinParams& p, uint32_t pos, uint32_t total, uint32_t base)
    {
        const uint32_t first = pos + 1u > p.window ? pos + 1u - p.window : 0u;
        end = static_cast<int32_t>(min(pos + 1u, total)) - 1 - static_cast<int32_t>(base);
        sinks = static_cast<int32_t>(p.sinks) - static_cast<int32_t>(base);
        low = static_cast<int32_t>(min(first, 0x7FFFFFFFu)) - static_cast<int32_t>(base);
    }
    __device__ __forceinline__ bool sees(int32_t y) const { return y <= end && (y < sinks || y >= low); }
};

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
        const WinMask m(p, pos, total, t0 + T::NS * g);
#pragma unroll
        for (uint32_t i = 0; i < T::NS; ++i) s[i] = m.sees(static_cast<int32_t>(i)) ? s[i] : NEG_INF;
    }
}

// log2 of a row's sum of 2^score from its maximum and sum; +inf (every weight 0)
// for a row with nothing to sum
__device__ __forceinline__ float win_lse(float m, float l) { return l == 0.0f ? __builtin_huge_valf() : m + __builtin_amdgcn_logf(l); }

// ---- window_prompt.hip
// a prompt's rows in one launch (16-bit caches); with p.lse, what k_win_sums needs
int win_prompt_launch(opure_dev* dev, const WinParams& p, uint32_t batch);
// weights += from the cache, the queries and p.lse; scratch of win_sums_bytes (n_heads, n_kv, rows, afmt and cap are read)
uint64_t win_sums_bytes(const opure_dev* dev, const WinParams& p, uint32_t batch);
uint64_t win_sums_workgroups(const opure_dev* dev, const WinParams& p, uint32_t batch);
int win_sums_launch(opure_dev* dev, const WinParams& p, uint32_t batch, float* scratch);

}  // namespace opure_win
