// ============================================================================
//  kv4_rows.hip -- attention of many query rows over the 4-bit paged cache.
// ============================================================================
#include "kv4_attn.h"

using namespace opure_kv4;

namespace {

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

// A workgroup takes 128 query rows (qi = j group + head) of a KV head, 32 a wave, over
// tiles of four pages (two past 128 channels) whose values the waves make from the codes
// once, each its page's, and share in LDS as operands: products are 32x32x16, S^T = K Q^T
// and O^T = V^T P^T.  A lane (q = lane % 32, h = lane / 32) holds of a page's scores the
// tokens 4 h .. 4 h + 3 and 8 + 4 h .. 11 + 4 h of row q, its operand P^T, and V of a
// page lies in LDS in that order of tokens.  Two stages: while one tile is computed the
// next one's values are made, each group's conversions between two products of K, and
// the words of the one after are on their way; a page's weights are made between the
// products of the page before, its values read a page ahead.  Left to itself the compiler
// takes few registers and waits for LDS before every product.
//   A tile that none of a wave's rows sees is computed all the same (two of a block's at
// most): with a branch round it and this order the outputs are copied twice a tile, 128
// moves beside 300 instructions, and 148 registers spill.
//   2,048 rows of 32 heads over 6,000 positions and themselves (8 KV heads of 128, bf16):
// 277 to 285 us by the device, 825 to 850 TFLOP/s of the 1,250 that a product of 8,192
// squared reaches; 291 to 298 in the compiler's order, 483 where each wave makes its own
// values.  Bound by the matrix units (44% of the clocks), the vector unit (63%) and LDS, of
// which products of 32 rows a wave read 56 bytes a clock of 128.  Two pages past 128
// channels, with a wave a SIMD and 512 registers, where the compiler's order is the better
// one (256 channels, 2,048 rows of 16 heads: 115 us, in this order 124).
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
    // K's and V's group g of tile i
    auto store_k = [&](uint32_t i, uint32_t g) {
        const uint32_t to = (lane >> 4 & 1u) * 32u + (mine & 1u) * 16u + (lane & 15u);
        // positions without a page: NaN keys for the rows that see them
        const half2_t sb = pair(pg < 0 ? 0x7E007E00u : ks[g]), sc = {sb[0], sb[0]}, ba = {sb[1], sb[1]};
        const u4v k = {values(bits.codes<0>(kw[g]), sc, ba), values(bits.codes<1>(kw[g]), sc, ba), values(bits.codes<2>(kw[g]), sc, ba), values(bits.codes<3>(kw[g]), sc, ba)};
        if (HD % 32 == 0 || g + 1u < NG || lane < 32u) k_at(i & 1u, mine >> 1, 2u * g + (lane >> 5))[to] = k;
    };
    auto store_v = [&](uint32_t i, uint32_t g) {
        const uint32_t x = lane >> 4, t = span.tile(i) * TT + 16u * mine + 4u * x, n = pg < 0 || t >= sq.total ? 0u : min(sq.total - t, 4u);
        const uint32_t m0 = n >= 2u ? 0xFFFFFFFFu : n == 1u ? 0xFFFFu : 0u, m1 = n >= 4u ? 0xFFFFFFFFu : n == 3u ? 0xFFFFu : 0u;
        // slots past the sequence and pages that are not there hold anything: 0
        const half2_t s0 = pair(vs[g][0] & m0), s1 = pair(vs[g][1] & m1), b0 = pair(vs[g][2] & m0), b1 = pair(vs[g][3] & m1);
        u2v* to = reinterpret_cast<u2v*>(v_at(i & 1u, mine, g) + (x & 1u) * 32u + (lane & 15u)) + (x >> 1);
        to[0] = u2v{values(bits.codes<0>(vw[g]), s0, b0), values(bits.codes<1>(vw[g]), s1, b1)};
        to[32] = u2v{values(bits.codes<2>(vw[g]), s0, b0), values(bits.codes<3>(vw[g]), s1, b1)};   // 16 channels on
    };
    auto store = [&](uint32_t i) {
        if (has_k)
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g) store_k(i, g);
        if (has_v)
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g) store_v(i, g);
    };

    // what is written on its two sides stays there
    auto apart = []() {
        if constexpr (!SPLIT) __builtin_amdgcn_sched_barrier(0);
    };
    f16_t o[NG];
    float m = NEG_INF, l = 0.0f;                            // the row's M; this lane's share of the sum
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
        if constexpr (!SPLIT)
        {
            fetch(min(first + 1u, last - 1u));
            entry(first + 2u);
        }
    }
    __syncthreads();
    for (uint32_t i = first; i < last; ++i)
    {
        const uint32_t stage = i & 1u, t0 = span.tile(i) * TT;
        if constexpr (SPLIT)
        {
            if (i + 1u < last) fetch(i + 1u);
            entry(i + 2u);
        }
        f16_t s[NP / 2u];
#pragma unroll
        for (uint32_t x = 0; x < NP / 2u; ++x)
#pragma unroll
            for (uint32_t y = 0; y < 16; ++y) s[x][y] = 0.0f;
        u4v k[2][NP / 2u];
        auto read_k = [&](uint32_t d) {
#pragma unroll
            for (uint32_t x = 0; x < NP / 2u; ++x) k[d & 1u][x] = k_at(stage, x, d)[lane];
        };
        read_k(0u);
        apart();
#pragma unroll
        for (uint32_t d = 0; d < 2u * NG; ++d)
        {
            if (d + 1u < KS) read_k(d + 1u);
            if (d < KS)
#pragma unroll
                for (uint32_t x = 0; x < NP / 2u; ++x)
#pragma unroll
                    for (uint32_t z = 0; z < QT; ++z) s[x] = mfma_32(k[d & 1u][x], q[z][d], s[x]);
            if constexpr (!SPLIT)
            {
                if (d & 1u) store_v(i + 1u, d >> 1);
                else store_k(i + 1u, d >> 1);
            }
            apart();
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
        if constexpr (!SPLIT)
        {
            if (i + 2u < last) fetch(i + 2u);
            entry(i + 3u);
        }
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
        const bool grown = has_grown(m, mx, c);
        if (__any(grown))
        {
            const float a = grow(grown, mx, c, m, l);
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g)
#pragma unroll
                for (uint32_t y = 0; y < 16; ++y) o[g][y] = __fmul_rn(o[g][y], a);
        }
        const float down = m == NEG_INF ? 0.0f : __fsub_rn(SHIFT, m);
        u4v hi[2], lo[2], v[2][NG];
        auto read_v = [&](uint32_t x) {
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g) v[x & 1u][g] = v_at(stage, x, g)[lane];
        };
        // two of a page's eight weights
        auto weigh = [&](uint32_t x, uint32_t y) {
            const float e0 = __builtin_amdgcn_exp2f(__fmaf_rn(s[x >> 1][8u * (x & 1u) + 2u * y], c, down));
            const float e1 = __builtin_amdgcn_exp2f(__fmaf_rn(s[x >> 1][8u * (x & 1u) + 2u * y + 1u], c, down));
            l += e0;
            l += e1;
            const uint32_t w = win_pack<OPURE_A_F16>(e0, e1);
            hi[x & 1u][y] = w;
            if constexpr (REST) lo[x & 1u][y] = win_pack<OPURE_A_F16>(__fsub_rn(e0, win_low<OPURE_A_F16>(w)), __fsub_rn(e1, win_high<OPURE_A_F16>(w)));
        };
        read_v(0u);
        apart();
#pragma unroll
        for (uint32_t y = 0; y < 4; ++y) weigh(0u, y);
#pragma unroll
        for (uint32_t x = 0; x < NP; ++x)
        {
            if (x + 1u < NP) read_v(x + 1u);
            apart();
#pragma unroll
            for (uint32_t g = 0; g < std::max(NG, 4u); ++g)
            {
                if (g < NG)
                {
                    if constexpr (REST) o[g] = mfma_32(v[x & 1u][g], lo[x & 1u], o[g]);
                    o[g] = mfma_32(v[x & 1u][g], hi[x & 1u], o[g]);
                }
                if (x + 1u < NP && g < 4u) weigh(x + 1u, g);
                apart();
            }
        }
        if constexpr (SPLIT)
        {
            if (i + 1u < last) store(i + 1u);
        }
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
            p.part_ml[at * 2u] = m;
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

}  // namespace

namespace opure_kv4 {

int kv4_rows_launch(opure_dev* dev, const WinParams& p, uint32_t wgs)
{
    auto by_head = [&](auto af) {
        return win_by_head(p.hd, [&](auto h) {
            constexpr int AF = decltype(af)::value, HD = decltype(h)::value;
            static std::atomic<uint64_t> done{0};
            auto* kernel = &k_kv4_rows<AF, HD>;
            const int rc = win_lds(dev, reinterpret_cast<const void*>(kernel), rows_lds<HD>(), done);
            if (rc) return rc;
            OPURE_LAUNCH(dev, kernel, dim3(wgs), dim3(256), rows_lds<HD>(), p);
            OPURE_LAUNCH_CHECK("k_kv4_rows");
            return OPURE_OK;
        });
    };
    return p.afmt == OPURE_A_F32   ? by_head(std::integral_constant<int, OPURE_A_F32>{})
           : p.afmt == OPURE_A_F16 ? by_head(std::integral_constant<int, OPURE_A_F16>{})
                                   : by_head(std::integral_constant<int, OPURE_A_BF16>{});
}

}  // namespace opure_kv4
