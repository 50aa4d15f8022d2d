// ============================================================================
//  kv4_one.hip -- attention over the 4-bit paged cache where a sequence is short
//  for what a launch costs: one workgroup a sequence, KV head and block of query
//  rows, and no second launch that joins.
// ============================================================================
#include "kv4_attn.h"

using namespace opure_kv4;

namespace {

// waves of a workgroup: 16 where their registers (128 a lane) and outputs in LDS are there
template <int HD, int NT>
constexpr uint32_t one_waves() { return HD <= 64 && NT == 1 ? 16u : 8u; }

// A workgroup takes all tiles that a sequence's rows see, for 16 NT query rows of a KV
// head, a wave every W-th; the waves are merged in LDS and the rows written.  Bound by the
// launch and round trips to memory: one row of 8 KV heads of 64 over 100 positions 4.8 us,
// over 300 5.9 (in two launches 8.2), of 128 5.4 and 6.4; 32 sequences of 300 of 128 7.1.
template <int AF, int HD, int NT, bool ONCE>
__global__ __launch_bounds__((64 * one_waves<HD, NT>())) void k_kv4_one(WinParams p)
{
    constexpr uint32_t DT = HD / 16u, W = one_waves<HD, NT>();
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ uint32_t again[NT];                         // rows that are not finite
    f4_t* cacc = reinterpret_cast<f4_t*>(lds);                            // [wave][DT][NT][64]
    float* cml = reinterpret_cast<float*>(lds + W * DT * NT * 64u * 16u);   // [wave][NT][16][2]
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t kh = blockIdx.x % p.n_kv, rest = blockIdx.x / p.n_kv, b = ONCE ? rest : rest / p.blocks, blk = ONCE ? 0u : rest - b * p.blocks;
    if (threadIdx.x < NT) again[threadIdx.x] = 0u;
    Kv4Wave<AF, HD, NT, ONCE, W> w(p, kh, blk * 16u * NT);
    w.seek(b);
    w.start(b, wave, w.span.n);
    w.run();
    w.leave(wave, cacc, cml);
    __syncthreads();
    auto row_of = [&](uint32_t qi) {
        const uint32_t j = qi / w.G;
        return (static_cast<uint64_t>(b) * p.rows + j) * p.n_heads + kh * w.G + (qi - j * w.G);
    };
    for (uint32_t u = wave; u < NT * DT; u += W)
    {
        const uint32_t n = u / DT, d = u - n * DT, qi = w.q0 + 16u * n + w.r;
        float M = NEG_INF, L = 0.0f;
#pragma unroll
        for (uint32_t x = 0; x < W; ++x) M = fmaxf(M, cml[((x * NT + n) * 16u + w.r) * 2u]);
        f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t x = 0; x < W; ++x)
        {
            const float f = __builtin_amdgcn_exp2f(__fsub_rn(cml[((x * NT + n) * 16u + w.r) * 2u], M == NEG_INF ? 0.0f : M));
            const f4_t v = cacc[((x * DT + d) * NT + n) * 64u + w.lane];
            L = __fmaf_rn(f, cml[((x * NT + n) * 16u + w.r) * 2u + 1u], L);
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y) acc[y] = __fmaf_rn(f, v[y], acc[y]);
        }
        if (qi >= w.Gq) continue;
        bool fine = true;
#pragma unroll
        for (uint32_t y = 0; y < 4; ++y)
        {
            acc[y] = L == 0.0f ? 0.0f : __fdiv_rn(acc[y], L);
            fine = fine && __builtin_isfinite(acc[y]);
        }
        if (!fine) atomicOr(&again[n], 1u << w.r);
        const uint64_t at = row_of(qi) * HD + 16u * d + 4u * w.g;
        if constexpr (AF == OPURE_A_F32)
        {
            float2* to = reinterpret_cast<float2*>(static_cast<float*>(p.out) + at);
            to[0] = float2{acc[0], acc[1]};
            to[1] = float2{acc[2], acc[3]};
        }
        else *reinterpret_cast<u2v*>(static_cast<uint16_t*>(p.out) + at) = u2v{win_pack<AF>(acc[0], acc[1]), win_pack<AF>(acc[2], acc[3])};
    }
    __syncthreads();
    // again position by position: a NaN among the values of a position that the row does not see meets weight 0 above
    float* const qs = reinterpret_cast<float*>(lds) + wave * 256u;
    for (uint32_t x = wave; x < 16u * NT; x += W)
    {
        if (!(again[x >> 4] >> (x & 15u) & 1u)) continue;
        const uint64_t row = row_of(w.q0 + x);
        __builtin_amdgcn_wave_barrier();
        for (uint32_t d = w.lane; d < HD; d += 64u) qs[d] = load_act<AF>(p.q, row * HD + d);
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float l, v[4];
        kv4_row(p, qs, b, kh, w.sq.ctx + (w.q0 + x) / w.G, w.sq.total, l, v);
#pragma unroll
        for (uint32_t y = 0; y < 4; ++y)
            if (w.lane + 64u * y < HD) store_act_rt(p.out, row * HD + w.lane + 64u * y, l == 0.0f ? 0.0f : __fdiv_rn(v[y], l), AF);
    }
}

}  // namespace

namespace opure_kv4 {

uint32_t kv4_one_waves(uint32_t hd, bool two) { return hd <= 64u && !two ? 16u : 8u; }

int kv4_one_launch(opure_dev* dev, const WinParams& p, uint32_t wgs)
{
    auto one = [&](auto af, auto h, auto nt, auto alone) {
        constexpr int AF = decltype(af)::value, HD = decltype(h)::value, NT = decltype(nt)::value;
        constexpr uint32_t W = one_waves<HD, NT>(), LDS = std::max(wave_lds<HD, NT, W>(), W * 1024u);
        static std::atomic<uint64_t> done{0};
        auto* kernel = &k_kv4_one<AF, HD, NT, decltype(alone)::value>;
        const int rc = win_lds(dev, reinterpret_cast<const void*>(kernel), LDS, done);
        if (rc) return rc;
        OPURE_LAUNCH(dev, kernel, dim3(wgs), dim3(64u * W), LDS, p);
        OPURE_LAUNCH_CHECK("k_kv4_one");
        return OPURE_OK;
    };
    typedef std::integral_constant<int, 1> One;
    auto by_head = [&](auto af) {
        return win_by_head(p.hd, [&](auto h) {
            if constexpr (decltype(h)::value <= 128)
            {
                if (p.two) return one(af, h, std::integral_constant<int, 2>{}, std::false_type{});
            }
            else if (p.blocks > 1u) return one(af, h, One{}, std::false_type{});
            return one(af, h, One{}, std::true_type{});
        });
    };
    return p.afmt == OPURE_A_F32   ? by_head(std::integral_constant<int, OPURE_A_F32>{})
           : p.afmt == OPURE_A_F16 ? by_head(std::integral_constant<int, OPURE_A_F16>{})
                                   : by_head(std::integral_constant<int, OPURE_A_BF16>{});
}

}  // namespace opure_kv4
