// ============================================================================
//  window_prompt.hip -- windowed attention of a prompt's rows, and the weights
//  that the cached positions got from many rows.
// ============================================================================
#include "window.h"

using namespace opure_win;

namespace {

typedef float f16_t __attribute__((ext_vector_type(16)));

template <int AF>
__device__ __forceinline__ f16_t mfma_32(u4v a, u4v b, f16_t c)
{
    if constexpr (AF == OPURE_A_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

constexpr uint32_t PT = 64;                                // positions a tile
template <int HD>
constexpr uint32_t prompt_k_pieces() { return PT * (HD / 8u + 1u); }   // a padded row a position
template <int HD>
constexpr uint32_t prompt_v_pieces() { return (HD + 31u) / 32u * 32u * (PT / 8u + 1u); }   // a padded row a channel
template <int HD>
constexpr uint32_t prompt_lds() { return 2u * (prompt_k_pieces<HD>() + prompt_v_pieces<HD>()) * 16u; }

// Many query rows: a workgroup takes 128 query rows (qi = j group + head) of a KV
// head, 32 a wave, over tiles of 64 positions that the four waves share in LDS,
// two stages deep, the next tile's loads in flight while one computes.  Products
// are 32x32x16: S^T = K Q^T with a lane (q = lane % 32, h = lane / 32) holding 32
// scores of one row, whose maximum and sum need one exchange between the halves;
// K rows lie in LDS in the order (positions with bits 2 and 3 exchanged) that
// makes a lane's scores 8 consecutive positions, its operand of O^T = V^T P^T.
//   A row's output is scaled to a new maximum only where that passes the old one
// by 2^8: the weights are then up to 2^8, which costs none of their bits.  A weight
// enters the product as two 16-bit numbers, as in k_win_split (2^-16 of it is lost in
// bf16, 2^-22 in fp16; the result's own rounding is 2^-8, 2^-11): the second product
// costs the 8B prompt 162 -> 209 us and the 1B one 18.1 -> 20.3, rounding the weights
// once left its results 1.4 times as far from the exact ones as one rounding at the
// end.  fp16 weights are held 2^6 higher, so that the smallest steps are small
// against the row's largest weight.
//   Bound by the matrix and vector units together, each busy in half of the clocks:
// 2,048 rows of 32 heads of 128 over 4,096 positions each take 208 us, 660 TFLOP/s of
// the formulas and 990 of the products done, where a library product of 8,192 x 8,192
// matrices reaches 1,133 to 1,160; 1,437 rows of 32 heads of 64 behind a window of 512,
// ten tiles a workgroup, 20.5 us.
//   KG 2 (a grid that does not give every SIMD two waves): eight waves, two for
// each 32 rows, one on the even tiles and one on the odd ones, merged at the end.
template <int AF, int HD, int KG>
__global__ __launch_bounds__(256 * KG) __attribute__((amdgpu_waves_per_eu(HD <= 128 ? 2 : 1))) void k_win_prompt(WinParams p)
{
    constexpr uint32_t KS = HD / 16u, DT = (HD + 31u) / 32u, P = HD / 8u, KROW = P + 1u, VROW = PT / 8u + 1u;
    constexpr uint32_t N = 8u * HD, NP = (N + 255u) / 256u;   // 16-byte pieces of a tile's K (and of its V); a thread's
    constexpr float UP = AF == OPURE_A_F16 ? 6.0f : 0.0f;
    extern __shared__ __align__(16) uint8_t lds[];
    const uint32_t kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0u;   // takes tiles kg, kg + KG, ...
    u4v* const kt = reinterpret_cast<u4v*>(lds) + kg * (prompt_lds<HD>() / 16u);
    u4v* const vt = kt + 2u * prompt_k_pieces<HD>();
    const uint32_t G = p.n_heads / p.n_kv, Gq = G * p.rows, nblk = (Gq + 127u) / 128u;
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, b = rest / nblk;
    const uint32_t q0 = (nblk - 1u - (rest - b * nblk)) * 128u;   // the rows that see most first
    const uint32_t tid = threadIdx.x & 255u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63u, h = lane >> 5, r = lane & 31u;
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    const WinSeq sq = win_seq(p, p.seq_len[b]);
    const uint32_t j0 = q0 / G, j1 = min(q0 + 127u, Gq - 1u) / G;
    const WinSpan span = win_span<PT>(p, sq, sq.ctx + j0, sq.ctx + j1 + 1u);
    // the wave's rows
    const uint32_t w0 = min(q0 + 32u * wave, Gq - 1u), w1 = min(q0 + 32u * wave + 31u, Gq - 1u), qi = min(w0 + r, Gq - 1u);
    const uint32_t j = qi / G, pos = sq.ctx + j, pos0 = sq.ctx + w0 / G, pos1 = sq.ctx + w1 / G;
    const uint64_t row = (static_cast<uint64_t>(b) * p.rows + j) * p.n_heads + kh * G + (qi - j * G);
    // scores in powers of two are c times the products: c >= 0, its sign goes to Q, and with c = 0 Q is 0 (NaN where it is
    // not finite: 0 times that)
    const float c = p.scale == 0.0f ? 1.0f : __fmul_rn(__builtin_fabsf(p.scale), 1.44269504088896340736f);
    constexpr uint32_t EXP = AF == OPURE_A_F16 ? 0x7C00u : 0x7F80u, QNAN = AF == OPURE_A_F16 ? 0x7E00u : 0x7FC0u;
    u4v q[KS];
#pragma unroll
    for (uint32_t s = 0; s < KS; ++s)
    {
        q[s] = *reinterpret_cast<const u4v*>(static_cast<const uint8_t*>(p.q) + row * (HD * 2u) + (2u * s + h) * 16u);
        const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
        {
            const uint32_t x = q[s][i], none = ((x & EXP) == EXP ? QNAN : 0u) | ((x >> 16 & EXP) == EXP ? QNAN << 16 : 0u);
            q[s][i] = p.scale == 0.0f ? none : x ^ flip;
        }
    }
    const uint64_t plane = static_cast<uint64_t>(OPURE_PAGE_SIZE) * HD * 2u, page_bytes = 2ull * p.n_kv * plane;
    const uint8_t* base = static_cast<const uint8_t*>(p.pool) + static_cast<uint64_t>(p.layer) * p.n_pages * page_bytes + kh * plane;
    const uint64_t vofs = p.n_kv * plane;

    // the loads of the next DEPTH tiles, a set of registers each
    constexpr uint32_t DEPTH = HD <= 96 ? 2u : 1u;
    u4v kr[DEPTH][NP], vr[DEPTH][NP];
    int32_t pe[NP], cur[DEPTH][NP];
    auto entries = [&](uint32_t i) {
        const uint32_t tile = span.tile(min(i * KG + kg, span.n - 1u));
#pragma unroll
        for (uint32_t u = 0; u < NP; ++u) pe[u] = pt[min(tile * 4u + (u * 256u + tid) / (2u * HD), p.max_pages - 1u)];
    };
    auto load = [&](uint32_t i, auto set) {
        constexpr uint32_t D = decltype(set)::value;
        const uint32_t tile = span.tile(i * KG + kg);
#pragma unroll
        for (uint32_t u = 0; u < NP; ++u)
        {
            const uint32_t e = u * 256u + tid, pg = e / (2u * HD);
            if (N % 256u != 0u && e >= N) continue;
            cur[D][u] = (tile * 4u + pg) * OPURE_PAGE_SIZE < sq.total && static_cast<uint32_t>(pe[u]) < p.n_pages ? pe[u] : -1;
            const uint8_t* at = base + static_cast<uint64_t>(cur[D][u] < 0 ? 0u : static_cast<uint32_t>(cur[D][u])) * page_bytes + (e - pg * 2u * HD) * 16u;
            kr[D][u] = *reinterpret_cast<const u4v*>(at);
            vr[D][u] = *reinterpret_cast<const u4v*>(at + vofs);
        }
    };
    auto store = [&](uint32_t i, auto set) {
        constexpr uint32_t D = decltype(set)::value;
        const uint32_t t0 = span.tile(i * KG + kg) * PT;
        u4v* k = kt + (i & 1u) * prompt_k_pieces<HD>();
        u4v* v = vt + (i & 1u) * prompt_v_pieces<HD>();
        const uint32_t nan = AF == OPURE_A_F16 ? 0x7E007E00u : 0x7FC07FC0u;
        const bool tail = t0 + PT > sq.total;
#pragma unroll
        for (uint32_t u = 0; u < NP; ++u)
        {
            const uint32_t e = u * 256u + tid, pg = e / (2u * HD), w = e - pg * 2u * HD;
            if (N % 256u != 0u && e >= N) continue;
            // positions without a page: NaN keys for the rows that see them, no values;
            // slots past the sequence hold anything: values 0
            u4v x = vr[D][u];
            const uint32_t tv = t0 + pg * OPURE_PAGE_SIZE + (w & 1u) * 8u;
            if (tail) x = win_tail<AF>(x, tv < sq.total ? sq.total - tv : 0u);
            x = cur[D][u] < 0 ? u4v{0u, 0u, 0u, 0u} : x;
            const uint32_t t = e / P, at = (t & ~12u) | ((t & 4u) << 1) | ((t & 8u) >> 1);
            k[at * KROW + e % P] = cur[D][u] < 0 ? u4v{nan, nan, nan, nan} : kr[D][u];
            v[(w >> 1) * VROW + pg * 2u + (w & 1u)] = x;
        }
    };

    f16_t o[DT];
    float m = NEG_INF, l = 0.0f;
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) o[d][i] = 0.0f;
    if constexpr (HD % 32 != 0)
    {
        // the last channel tile's upper half is not there: zeros
        for (uint32_t e = tid; e < 2u * 16u * VROW; e += 256u)
            vt[(e / (16u * VROW)) * prompt_v_pieces<HD>() + HD * VROW + e % (16u * VROW)] = u4v{0u, 0u, 0u, 0u};
    }
    typedef std::integral_constant<uint32_t, 0> First;
    typedef std::integral_constant<uint32_t, DEPTH - 1u> Second;
    const uint32_t turns = (span.n + KG - 1u) / KG, own = (span.n + KG - 1u - kg) / KG;   // the workgroup's, and this half's tiles
    if (own)
    {
        entries(0u);
        load(0u, First{});
        entries(1u);
        if (DEPTH > 1u && own > 1u)
        {
            load(1u, Second{});
            entries(2u);
        }
    }
    auto tile = [&](uint32_t i, auto set) {
        if (KG == 1 || i < own) store(i, set);
        __syncthreads();
        if (KG > 1 && i >= own) return;
        if (i + DEPTH < own)
        {
            load(i + DEPTH, set);
            entries(i + DEPTH + 1u);
        }
        const uint32_t t0 = span.tile(i * KG + kg) * PT;
        // nothing of the tile that a row of the wave sees
        if (t0 > pos1 || (t0 >= p.sinks && t0 + PT - 1u + p.window <= pos0)) return;
        const u4v* k = kt + (i & 1u) * prompt_k_pieces<HD>();
        const u4v* v = vt + (i & 1u) * prompt_v_pieces<HD>();
        f16_t s[2];
        // the reads of the next key operand between the products of this one, and the products ahead of the other
        // waves' vector work (with one product a weight: 8B prompt 183.5 -> 180.9 us, 1B 18.3 -> 18.1)
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t)
        {
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) s[t][x] = 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < KS; ++x) s[t] = mfma_32<AF>(k[(32u * t + r) * KROW + 2u * x + h], q[x], s[t]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, KS, 0);
#pragma unroll
        for (uint32_t x = 0; x < KS; ++x)
        {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, KS, 0);
        __builtin_amdgcn_s_setprio(0);
        if (t0 + PT > min(pos0 + 1u, sq.total) || !(t0 + PT <= p.sinks || t0 + p.window > pos1))
        {
            const WinMask mask(p, pos, sq.total, t0 + 8u * h);
#pragma unroll
            for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
                for (uint32_t x = 0; x < 16; ++x)
                    s[t][x] = mask.sees(static_cast<int32_t>(32u * t + 16u * (x >> 3) + (x & 7u))) ? s[t][x] : NEG_INF;
        }
        float mx = s[0][0];
#pragma unroll
        for (uint32_t x = 1; x < 32; ++x) mx = fmaxf(mx, s[x >> 4][x & 15u]);
        mx = __fmul_rn(max_xor32(mx), c);
        if (__any(mx > m + 8.0f))
        {
            const float mn = fmaxf(m, mx), a = __builtin_amdgcn_exp2f(__fsub_rn(m, mn == NEG_INF ? 0.0f : mn));
            l = __fmul_rn(l, a);
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
                for (uint32_t x = 0; x < 16; ++x) o[d][x] = __fmul_rn(o[d][x], a);
            m = mn;
        }
        const float ms = m == NEG_INF ? 0.0f : m - UP;
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
        {
            u4v w, rest;
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
            {
                const float s0 = s[u >> 1][8u * (u & 1u) + 2u * x], s1 = s[u >> 1][8u * (u & 1u) + 2u * x + 1u];
                const float e0 = __builtin_amdgcn_exp2f(__fmaf_rn(s0, c, -ms)), e1 = __builtin_amdgcn_exp2f(__fmaf_rn(s1, c, -ms));
                sum[0] += e0;
                sum[1] += e1;
                w[x] = win_pack<AF>(e0, e1);
                rest[x] = win_pack<AF>(__fsub_rn(e0, win_low<AF>(w[x])), __fsub_rn(e1, win_high<AF>(w[x])));
            }
            u4v vx[DT];
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) vx[d] = v[(32u * d + r) * VROW + 2u * u + h];
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) o[d] = mfma_32<AF>(vx[d], rest, o[d]);
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) o[d] = mfma_32<AF>(vx[d], w, o[d]);
        }
        l += sum[0] + sum[1];                              // this half's share
        // the next 16 positions' weights between the products of these (1B prompt 21.4 -> 20.3 us, 8B the same)
        __builtin_amdgcn_sched_group_barrier(0x002, 40, 0);
#pragma unroll
        for (uint32_t x = 0; x < 6u * DT; ++x)
        {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 20u / DT, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2u * DT, 0);
    };
    for (uint32_t i = 0; i < turns; i += DEPTH)
    {
        tile(i, First{});
        if (DEPTH > 1u && i + 1u < turns) tile(i + 1u, Second{});
    }
    if constexpr (KG > 1)
    {
        // the odd tiles' results to the waves of the even ones: a lane hands over its own registers
        __syncthreads();
        f4_t* give = reinterpret_cast<f4_t*>(lds) + wave * (4u * DT + 1u) * 64u + lane;
        if (kg)
        {
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) give[(4u * d + x) * 64u] = f4_t{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
            give[4u * DT * 64u] = f4_t{m, l, 0.0f, 0.0f};
        }
        __syncthreads();
        if (!kg)
        {
            const f4_t ml = give[4u * DT * 64u];
            const float mn = fmaxf(m, ml[0]), ms = mn == NEG_INF ? 0.0f : mn;
            const float a = __builtin_amdgcn_exp2f(__fsub_rn(m, ms)), c2 = __builtin_amdgcn_exp2f(__fsub_rn(ml[0], ms));
            l = __fmaf_rn(ml[1], c2, __fmul_rn(l, a));
            m = mn;
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x)
                {
                    const f4_t v = give[(4u * d + x) * 64u];
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) o[d][4 * x + k] = __fmaf_rn(v[k], c2, __fmul_rn(o[d][4 * x + k], a));
                }
        }
    }
    l = add_xor32(l);
    const bool mine = kg == 0u && q0 + 32u * wave + r < Gq;
    if (p.lse && h == 0u && mine) p.lse[(static_cast<uint64_t>(b) * p.n_kv + kh) * Gq + qi] = win_lse(m - UP, l);
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    bool fine = true;
    typedef uint32_t u2v __attribute__((ext_vector_type(2)));
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
        for (uint32_t x = 0; x < 16; x += 4)
        {
            const uint32_t ch = 32u * d + 2u * x + 4u * h;
            if (HD % 32 != 0 && ch >= HD) continue;
            float y[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
            {
                y[k] = __fmul_rn(o[d][x + k], inv);
                fine = fine && __builtin_isfinite(y[k]);
            }
            if (mine)
                *reinterpret_cast<u2v*>(static_cast<uint8_t*>(p.out) + (row * HD + ch) * 2u) = u2v{win_pack<AF>(y[0], y[1]), win_pack<AF>(y[2], y[3])};
        }
    // rows that are not finite, position by position (k_win_join's reason)
    uint64_t bad = __ballot(!fine && mine);
    bad = (bad | bad >> 32) & 0xFFFFFFFFull;
    __syncthreads();                                       // the stages are done with
    float* qs = reinterpret_cast<float*>(lds) + wave * 256u;   // the even half's: the others have no row
    while (bad)
    {
        const uint32_t x = static_cast<uint32_t>(__builtin_ctzll(bad));
        bad &= bad - 1u;
        const uint32_t qx = w0 + x, jx = qx / G;
        const uint64_t rx = ((static_cast<uint64_t>(b) * p.rows + jx) * p.n_heads + kh * G + (qx - jx * G)) * HD;
        for (uint32_t d = lane; d < HD; d += 64u) qs[d] = load_act_rt(p.q, rx + d, p.afmt);
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float mm, ll, oo[4];
        win_row(p, qs, b, kh, sq.ctx + jx, sq.total, mm, ll, oo);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (lane + 64u * i < HD) store_act_rt(p.out, rx + lane + 64u * i, ll == 0.0f ? 0.0f : __fdiv_rn(oo[i], ll), p.afmt);
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Weights from many rows: a workgroup takes 64 positions (32 of an fp32 cache) of
// a (sequence, KV head) and a chunk of query rows, its four waves every
// fourth block of 16 of those rows that see one of the positions.  A wave holds
// the positions' keys as operands, computes the block's scores again and adds
// 2^(score - lse) to a sum a lane and position; the lanes' and waves' sums are
// added in order.
//   With more than one chunk each leaves its sums in a place of its own, and
// k_win_add adds them in order: the first positions of a prompt are seen by all of
// its rows, which one workgroup took 30 us to walk through (1,024 rows of the 1B
// shape; 16 in chunks).  Bound there by its first loads and by the exponentials,
// 16 clocks each on a SIMD.  Whole calls with chunks of 512, 1,024, 1,536, 2,048
// and 4,096: that prompt 41.4, 38.9, 39.3, 40.7, 50.0 us; 2,048 rows 90.5, 90.0,
// 82.5, 88.8, 89.9; 2,048 rows of 128 channels behind a window of 4,096 414, 386,
// 375, 390, 364.  Where chunks of 1,536 do not give every CU a workgroup, which
// walks its rows alone, they are of 512 (whole calls with 1,536 / 512: 2,008 rows of
// 4 heads of 64 behind a window of 20 34.8 / 24.9, 512 rows of 32 heads 30.0 / 24.9,
// 400 of 12 heads of 112 in fp32 54.8 / 41.9; but with 400 workgroups 66.3 / 75.0).
uint32_t sums_chunk(const opure_dev* dev, const WinParams& p, uint32_t batch)
{
    const uint32_t Gq = p.n_heads / p.n_kv * p.rows, tile = p.afmt == OPURE_A_F32 ? 32u : 64u;
    const uint64_t wgs = static_cast<uint64_t>(p.n_kv) * batch * ((p.cap + tile - 1u) / tile) * ((Gq + 1535u) / 1536u);
    return wgs <= static_cast<uint32_t>(dev->n_cu > 0 ? dev->n_cu : 256) ? 512u : 1536u;
}

// rows [ja, jz) of a chunk that see a position of [t0, t0 + n)
__device__ __forceinline__ void sums_rows(const WinParams& p, const WinSeq& sq, uint32_t G, uint32_t chunk, uint32_t t0, uint32_t n,
                                          uint32_t& qa, uint32_t& qz)
{
    const uint32_t ja = t0 > sq.ctx ? t0 - sq.ctx : 0u;
    const uint32_t jz = t0 < p.sinks ? p.rows : t0 + n - 1u + p.window > sq.ctx ? min(p.rows, t0 + n - 1u + p.window - sq.ctx) : 0u;
    qa = max(ja * G, chunk * p.sum_rows);
    qz = min(jz * G, (chunk + 1u) * p.sum_rows);
    if (t0 >= sq.total) qz = 0u;
}

constexpr uint32_t SUM_WAVES = 4;

template <int AF, int HD>
__global__ __launch_bounds__(64 * SUM_WAVES) __attribute__((amdgpu_waves_per_eu(HD <= 64 && AF != OPURE_A_F32 ? 4 : HD <= 128 ? 2 : 1))) void k_win_sums(WinParams p)
{
    typedef WinTile<AF, HD> T;
    constexpr uint32_t NS = T::NS, TILE = 2u * T::TT;
    __shared__ float part[SUM_WAVES][TILE];
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, chunk = rest % p.parts, rest2 = rest / p.parts;
    const uint32_t b = rest2 % p.batch, tile = rest2 / p.batch;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t G = p.n_heads / p.n_kv, Gq = G * p.rows, t0 = tile * TILE;
    const int32_t* pt = p.page_table + static_cast<uint64_t>(b) * p.max_pages;
    // the length and the tile's page entries (a lane each) in one round trip
    const int32_t len = p.seq_len[b];
    const int32_t entries = pt[min(t0 / OPURE_PAGE_SIZE + (lane & (2u * T::NB - 1u)), p.max_pages - 1u)];
    asm volatile("" ::: "memory");
    const WinSeq sq = win_seq(p, len);
    uint32_t qa, qz;
    sums_rows(p, sq, G, chunk, t0, TILE, qa, qz);
    if (qa >= qz) return;                                  // whole workgroup
    const uint64_t page_bytes = 2ull * p.n_kv * T::PB;
    const uint8_t* base = static_cast<const uint8_t*>(p.pool) + static_cast<uint64_t>(p.layer) * p.n_pages * page_bytes + static_cast<uint64_t>(kh) * T::PB;
    T tl[2];
    bool whole = t0 + TILE <= sq.total;
#pragma unroll
    for (uint32_t x = 0; x < 2; ++x)
    {
        int32_t pg[2];
#pragma unroll
        for (uint32_t y = 0; y < T::NB; ++y)
        {
            const int32_t e = __builtin_amdgcn_readlane(entries, x * T::NB + y);
            pg[y] = t0 + x * T::TT + y * OPURE_PAGE_SIZE < sq.total && static_cast<uint32_t>(e) < p.n_pages ? e : -1;
        }
        if (T::NB == 1u) pg[1] = pg[0];
        auto at = [&](int32_t e) { return base + static_cast<uint64_t>(e < 0 ? 0u : static_cast<uint32_t>(e)) * page_bytes; };
        tl[x].template load_k<false>(at(pg[0]), at(pg[1]), r, g);
        const uint32_t nan = AF == OPURE_A_F32 ? 0x7FC00000u : AF == OPURE_A_F16 ? 0x7E007E00u : 0x7FC07FC0u;
        const bool gone = (T::NB > 1u && r >= 8u ? pg[1] : pg[0]) < 0;
        whole = whole && pg[0] >= 0 && pg[1] >= 0;
        if (pg[0] < 0 || pg[1] < 0)
#pragma unroll
        for (uint32_t t = 0; t < T::NB; ++t)
#pragma unroll
            for (uint32_t s = 0; s < T::KS; ++s) tl[x].k[t][s] = gone ? u4v{nan, nan, nan, nan} : tl[x].k[t][s];
    }
    // the keys have arrived: the loop's waits are for the queries alone
#pragma unroll
    for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
        for (uint32_t t = 0; t < T::NB; ++t)
#pragma unroll
            for (uint32_t s = 0; s < T::KS; ++s) asm volatile("" : "+v"(tl[x].k[t][s]));
    const float c = __fmul_rn(p.scale, 1.44269504088896340736f);
    float sum[2][NS];
#pragma unroll
    for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
        for (uint32_t y = 0; y < NS; ++y) sum[x][y] = 0.0f;
    const float* lse = p.lse + (static_cast<uint64_t>(b) * p.n_kv + kh) * Gq;
    // two blocks of rows a turn, the next turn's on their way (one where their operands are large)
    constexpr uint32_t BLK = HD <= 128 ? 2u : 1u, EACH = 16u * SUM_WAVES, STEP = EACH * BLK;
    u4v q[BLK][T::KS], nq[BLK][T::KS];
    float ls[BLK], nls[BLK];
    uint32_t jr[BLK], njr[BLK];
    auto fetch = [&](uint32_t q0, u4v (&to)[T::KS], float& l, uint32_t& j) {
        const uint32_t qi = min(q0 + r, Gq - 1u);
        j = qi / G;
        win_load_q<AF, HD>(p, (static_cast<uint64_t>(b) * p.rows + j) * p.n_heads + kh * G + (qi - j * G), g, to);
        l = lse[qi];
    };
    uint32_t q0 = qa + 16u * wave;
    if (q0 < qz)
#pragma unroll
        for (uint32_t u = 0; u < BLK; ++u) fetch(q0 + EACH * u, q[u], ls[u], jr[u]);
    for (; q0 < qz; q0 += STEP)
    {
        if (q0 + STEP < qz)
#pragma unroll
            for (uint32_t u = 0; u < BLK; ++u) fetch(q0 + STEP + EACH * u, nq[u], nls[u], njr[u]);
#pragma unroll
        for (uint32_t u = 0; u < BLK; ++u)
        {
            const uint32_t qb = q0 + EACH * u;
            if (qb >= qz) break;
            const uint32_t p0 = sq.ctx + qb / G, p1 = sq.ctx + min(qb + 15u, Gq - 1u) / G;
            const bool full = whole && t0 + TILE <= p0 + 1u && (t0 + TILE <= p.sinks || t0 + p.window > p1);
            const float of_row = qb + r < qz ? ls[u] : __builtin_huge_valf();   // a row past the last: weight 0
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x)
            {
                float s[NS];
#pragma unroll
                for (uint32_t t = 0; t < T::NB; ++t)
                {
                    f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (uint32_t k = 0; k < T::KS; ++k) acc = win_mfma<AF>(tl[x].k[t][k], q[u][k], acc);
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) s[4u * t + i] = __builtin_amdgcn_exp2f(__fmaf_rn(acc[i], c, -of_row));
                }
                if (!full)
                {
                    const WinMask m(p, sq.ctx + jr[u], sq.total, t0 + x * T::TT + NS * g);
#pragma unroll
                    for (uint32_t y = 0; y < NS; ++y) s[y] = m.sees(static_cast<int32_t>(y)) ? s[y] : 0.0f;
                }
#pragma unroll
                for (uint32_t y = 0; y < NS; ++y) sum[x][y] += s[y];
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < BLK; ++u)
        {
#pragma unroll
            for (uint32_t k = 0; k < T::KS; ++k) q[u][k] = nq[u][k];
            ls[u] = nls[u];
            jr[u] = njr[u];
        }
    }
#pragma unroll
    for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
        for (uint32_t y = 0; y < NS; ++y)
        {
            const float v = row16_sum(sum[x][y]);
            if (r == 0u) part[wave][x * T::TT + NS * g + y] = v;
        }
    __syncthreads();
    const uint32_t t = t0 + threadIdx.x;
    if (threadIdx.x >= TILE || t >= sq.total) return;
    float v = part[0][threadIdx.x];
#pragma unroll
    for (uint32_t w = 1; w < SUM_WAVES; ++w) v += part[w][threadIdx.x];
    if (p.parts > 1u)
    {
        p.part_acc[(static_cast<uint64_t>(b * p.n_kv + kh) * p.parts + chunk) * p.cap + t] = v;
        return;
    }
    // seen by a row: by the first at or past the position, if by any
    const uint32_t first = t > sq.ctx ? t - sq.ctx : 0u;
    if (first >= p.rows || !win_sees(p, sq.ctx + first, t)) return;
    p.weights[b * p.weights_batch_stride + static_cast<uint64_t>(kh) * p.weights_stride + t] += v;
}

// the chunks' sums, a thread a position
template <uint32_t TILE>
__global__ __launch_bounds__(256) void k_win_add(WinParams p)
{
    const uint32_t G = p.n_heads / p.n_kv, kh = blockIdx.y, b = blockIdx.z, t = blockIdx.x * 256u + threadIdx.x;
    const WinSeq sq = win_seq(p, p.seq_len[b]);
    if (t >= sq.total) return;
    const uint32_t first = t > sq.ctx ? t - sq.ctx : 0u;
    if (first >= p.rows || !win_sees(p, sq.ctx + first, t)) return;
    const float* part = p.part_acc + static_cast<uint64_t>(b * p.n_kv + kh) * p.parts * p.cap + t;
    float* to = p.weights + b * p.weights_batch_stride + static_cast<uint64_t>(kh) * p.weights_stride + t;
    const float old = *to;
    float v = 0.0f;
#pragma unroll 4
    for (uint32_t chunk = 0; chunk < p.parts; ++chunk)
    {
        uint32_t qa, qz;
        sums_rows(p, sq, G, chunk, t / TILE * TILE, TILE, qa, qz);
        if (qa < qz) v += part[static_cast<uint64_t>(chunk) * p.cap];
    }
    *to = old + v;
}

}  // namespace

namespace opure_win {

int win_prompt_launch(opure_dev* dev, const WinParams& p, uint32_t batch)
{
    const uint32_t Gq = p.n_heads / p.n_kv * p.rows, wgs = p.n_kv * ((Gq + 127u) / 128u) * batch;
    // KG 1 against 2: 256 workgroups (1,024 causal rows) 24.8 against 20.4 us, 360 behind a window of 512 19.0 against
    // 25.7, 512 23.9 against 28.5 (512 causal ones 47.2 against 42.5)
    const bool two = wgs <= static_cast<uint32_t>(dev->n_cu > 0 ? dev->n_cu : 256);
    auto go = [&](auto af) {
        return win_by_head(p.hd, [&](auto h) {
            constexpr int AF = decltype(af)::value, HD = decltype(h)::value;
            auto run = [&](auto groups) {
                constexpr int KG = decltype(groups)::value;
                static std::atomic<uint64_t> done{0};
                const int rc = win_lds(dev, reinterpret_cast<const void*>(&k_win_prompt<AF, HD, KG>), KG * prompt_lds<HD>(), done);
                if (rc) return rc;
                OPURE_LAUNCH(dev, (k_win_prompt<AF, HD, KG>), dim3(wgs), dim3(256 * KG), KG * prompt_lds<HD>(), p);
                OPURE_LAUNCH_CHECK("k_win_prompt");
                return OPURE_OK;
            };
            if constexpr (HD <= 128)
                if (two) return run(std::integral_constant<int, 2>{});
            return run(std::integral_constant<int, 1>{});
        });
    };
    return p.afmt == OPURE_A_F16 ? go(std::integral_constant<int, OPURE_A_F16>{}) : go(std::integral_constant<int, OPURE_A_BF16>{});
}

uint64_t win_sums_bytes(const opure_dev* dev, const WinParams& p, uint32_t batch)
{
    const uint32_t rows = sums_chunk(dev, p, batch);
    const uint64_t chunks = (static_cast<uint64_t>(p.n_heads / p.n_kv) * p.rows + rows - 1u) / rows;
    return chunks > 1u ? static_cast<uint64_t>(batch) * p.n_kv * chunks * p.cap * 4u : 0u;
}

uint64_t win_sums_workgroups(const opure_dev* dev, const WinParams& p, uint32_t batch)
{
    const uint32_t rows = sums_chunk(dev, p, batch), tile = p.afmt == OPURE_A_F32 ? 32u : 64u;
    const uint64_t chunks = (static_cast<uint64_t>(p.n_heads / p.n_kv) * p.rows + rows - 1u) / rows;
    return static_cast<uint64_t>(p.n_kv) * batch * chunks * ((p.cap + tile - 1u) / tile);
}

int win_sums_launch(opure_dev* dev, const WinParams& p, uint32_t batch, float* scratch)
{
    WinParams s = p;
    s.batch = batch;
    s.sum_rows = sums_chunk(dev, p, batch);
    s.parts = (p.n_heads / p.n_kv * p.rows + s.sum_rows - 1u) / s.sum_rows;
    s.part_acc = scratch;
    const uint32_t tile = p.afmt == OPURE_A_F32 ? 32u : 64u;
    auto go = [&](auto af) {
        return win_by_head(p.hd, [&](auto h) {
            constexpr int AF = decltype(af)::value, HD = decltype(h)::value;
            OPURE_LAUNCH(dev, (k_win_sums<AF, HD>), dim3(p.n_kv * batch * s.parts * ((p.cap + tile - 1u) / tile)), dim3(64 * SUM_WAVES), 0, s);
            OPURE_LAUNCH_CHECK("k_win_sums");
            return OPURE_OK;
        });
    };
    const int rc = p.afmt == OPURE_A_F32   ? go(std::integral_constant<int, OPURE_A_F32>{})
                   : p.afmt == OPURE_A_F16 ? go(std::integral_constant<int, OPURE_A_F16>{})
                                           : go(std::integral_constant<int, OPURE_A_BF16>{});
    if (rc || s.parts == 1u) return rc;
    const dim3 grid((p.cap + 255u) / 256u, p.n_kv, batch);
    if (tile == 32u) OPURE_LAUNCH(dev, (k_win_add<32u>), grid, dim3(256), 0, s);
    else OPURE_LAUNCH(dev, (k_win_add<64u>), grid, dim3(256), 0, s);
    OPURE_LAUNCH_CHECK("k_win_add");
    return OPURE_OK;
}

}  // namespace opure_win
