// ============================================================================
//  append.hip -- rows of queries, keys and values that a program has computed
//  itself: queries and keys turned to their positions, keys and values written to
//  a layer of the paged cache, in the model's format or in 4 bits (kv4.h).
//
//  Row j of a sequence stands at position p = seq_len + j.  A pair (x, y) of
//  channels 2 i, 2 i + 1 becomes (x c - y s, x s + y c) with the model's cosine and
//  sine of row p, each product and sum rounded to fp32 as in the fused QKV product,
//  so the cache's bits are those that a verify step writes for the same numbers.
// ============================================================================
#include "kv4.h"

#include <type_traits>

using namespace opure_dev_math;
using namespace opure_kv4;

namespace {

struct AppendParams {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    void* pool;
    const int32_t* page_table;
    const int32_t* seq_len;
    const int32_t* row_count;
    const float* cos;
    const float* sin;
    uint64_t q_stride, k_stride, v_stride;   // elements between rows
    uint32_t heads, n_kv, hd, ng, rows, n_pages, max_pages, layer;
    uint32_t cap;                            // positions that may be written: min(max_ctx, the table's)
    uint32_t q_units, k_units, v_units;      // threads a row (q, k: 8 channels each), or a piece of a sequence's positions (v)
    uint32_t k_first;                        // the row's first thread of k: q_units to the next four, whose lanes share a group
    uint32_t per_head;                       // 2^32 / (a head's threads among the k_units), rounded up; q_units': q_per_head
    uint32_t q_per_head, v_per_head;
    uint32_t batch;
    uint32_t row_cols, v_cols;               // waves a row, a piece
    uint32_t pieces;                         // most pieces that a sequence's rows touch: pages, or quarters of one
    uint32_t v_waves;                        // waves of all pieces; the others are the rows'
    uint32_t* err;
};

typedef float f8_t __attribute__((ext_vector_type(8)));

// n / d for n < 2^24 and d < 256, by m = 2^32 / d rounded up: n (m d - 2^32) < 2^32
__device__ __forceinline__ uint32_t div_by(uint32_t n, uint32_t m) { return m ? __umulhi(n, m) : n; }

template <int F>
__device__ __forceinline__ f8_t load8(const void* base, uint64_t at)
{
    f8_t x;
    if constexpr (F == OPURE_A_F32)
    {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        const float4 a = p[0], b = p[1];
        x = f8_t{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    }
    else
    {
        const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            x[2 * i] = F == OPURE_A_F16 ? f16_to_f32(static_cast<uint16_t>(u[i])) : bits_f(u[i] << 16);
            x[2 * i + 1] = F == OPURE_A_F16 ? f16_to_f32(static_cast<uint16_t>(u[i] >> 16)) : bits_f(u[i] & 0xFFFF0000u);
        }
    }
    return x;
}

template <int F>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    return F == OPURE_A_F16 ? f32_to_f16(a) | static_cast<uint32_t>(f32_to_f16(b)) << 16
                            : f32_to_bf16(a) | static_cast<uint32_t>(f32_to_bf16(b)) << 16;
}

template <int F>
__device__ __forceinline__ void store8(void* base, uint64_t at, f8_t x)
{
    if constexpr (F == OPURE_A_F32)
    {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        p[0] = float4{x[0], x[1], x[2], x[3]};
        p[1] = float4{x[4], x[5], x[6], x[7]};
    }
    else
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
            uint4{pack2<F>(x[0], x[1]), pack2<F>(x[2], x[3]), pack2<F>(x[4], x[5]), pack2<F>(x[6], x[7])};
}

// channels d .. d + 7 of a head turned to position pos
__device__ __forceinline__ f8_t turn8(const AppendParams& p, f8_t x, uint32_t pos, uint32_t d)
{
    if (!p.cos) return x;
    const uint64_t at = static_cast<uint64_t>(pos) * (p.hd / 2u) + d / 2u;
    const float4 c = *reinterpret_cast<const float4*>(p.cos + at), s = *reinterpret_cast<const float4*>(p.sin + at);
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
    f8_t y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        y[2 * i] = __fsub_rn(__fmul_rn(x[2 * i], cc[i]), __fmul_rn(x[2 * i + 1], ss[i]));
        y[2 * i + 1] = __fadd_rn(__fmul_rn(x[2 * i], ss[i]), __fmul_rn(x[2 * i + 1], cc[i]));
    }
    return y;
}

// A sequence's rows: positions first .. end - 1 are written.
struct AppendSeq {
    uint32_t first, end;
    bool bad;                                // some of them cannot be
    __device__ __forceinline__ AppendSeq(const AppendParams& p, uint32_t b)
    {
        const int32_t len = p.seq_len[b];
        const uint32_t n = p.row_count ? min(static_cast<uint32_t>(max(p.row_count[b], 0)), p.rows) : p.rows;
        first = static_cast<uint32_t>(max(len, 0));
        const uint32_t all = len < 0 ? first : first + n;
        end = max(first, min(all, p.cap));
        bad = n > 0u && (len < 0 || all > p.cap);
    }
};

__device__ __forceinline__ int32_t append_page(const AppendParams& p, uint32_t b, uint32_t pos)
{
    const int32_t pg = p.page_table[static_cast<uint64_t>(b) * p.max_pages + pos / OPURE_PAGE_SIZE];
    if (pg >= 0 && static_cast<uint32_t>(pg) < p.n_pages) return pg;
    p.err[ERR_POSITION] = 1u;
    return -1;
}

// 8 channels of a key from d on to 4 bits: four lanes a group, of half a group the last two
// have no channels (`there`)
__device__ __forceinline__ void put_k4(const AppendParams& p, f8_t x, bool there, uint32_t pg, uint32_t h, uint32_t i, uint32_t slot)
{
    float lo = __builtin_huge_valf(), hi = -__builtin_huge_valf();
    bool bad = false;
    if (there)
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            bad = bad || !__builtin_isfinite(x[e]);
            x[e] = fminf(fmaxf(x[e], -MOST), MOST);
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
        }
    lo = fminf(lo, dpp_f<0xB1>(lo));
    lo = fminf(lo, dpp_f<0x4E>(lo));
    hi = fmaxf(hi, dpp_f<0xB1>(hi));
    hi = fmaxf(hi, dpp_f<0x4E>(hi));
    const uint64_t any = __ballot(bad);
    const Scale sc(lo, hi, (any >> (threadIdx.x & 60u) & 15u) != 0u);
    uint32_t w = 0;
    float c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = x[e];
    sc.codes(c);
    if (there)
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= static_cast<uint32_t>(c[e]) << (16 * (e & 1) + 4 * (e >> 1));
    uint8_t* block = static_cast<uint8_t*>(p.pool) + block_at(p.layer, p.n_pages, pg, p.n_kv, h, p.ng);
    reinterpret_cast<uint32_t*>(block)[((i & 3u) * 16u + slot) * p.ng + (i >> 2)] = w;
    if ((i & 3u) == 0u) reinterpret_cast<uint32_t*>(block + k_scales(p.ng))[slot * p.ng + (i >> 2)] = sc.scale_bits() | sc.base_bits() << 16;
}

// Two channels, c and c + 16 of group g (`both`: the second is there), of the tokens t0 .. t0 + 3 to 4
// bits: sixteen lanes a group.  Tokens outside lo .. hi - 1 keep theirs.
__device__ __forceinline__ void put_v4(const AppendParams& p, const float (&x)[4][2], bool both, uint32_t pg, uint32_t h, uint32_t g, uint32_t c,
                                       uint32_t t0, uint32_t lo, uint32_t hi)
{
    uint8_t* block = static_cast<uint8_t*>(p.pool) + block_at(p.layer, p.n_pages, pg, p.n_kv, h, p.ng);
    const uint32_t j = t0 / 4u % 4u;
    uint32_t* to = reinterpret_cast<uint32_t*>(block + v_codes(p.ng)) + (j * 16u + c) * p.ng + g;
    uint16_t* sb = reinterpret_cast<uint16_t*>(block + v_scales(p.ng)) + (j * p.ng + g) * 8u;
    uint32_t w = 0, mine = 0;
#pragma unroll
    for (uint32_t t = 0; t < 4; ++t)
    {
        const bool bad = !__builtin_isfinite(x[t][0]) || !__builtin_isfinite(x[t][1]);
        const float y0 = fminf(fmaxf(x[t][0], -MOST), MOST), y1 = fminf(fmaxf(x[t][1], -MOST), MOST);
        float mn = fminf(y0, y1), mx = fmaxf(y0, y1);
        mn = fminf(mn, dpp_f<0xB1>(mn));
        mn = fminf(mn, dpp_f<0x4E>(mn));
        mn = fminf(mn, dpp_f<0x141>(mn));
        mn = fminf(mn, dpp_f<0x140>(mn));
        mx = fmaxf(mx, dpp_f<0xB1>(mx));
        mx = fmaxf(mx, dpp_f<0x4E>(mx));
        mx = fmaxf(mx, dpp_f<0x141>(mx));
        mx = fmaxf(mx, dpp_f<0x140>(mx));
        const Scale sc(mn, mx, (__ballot(bad) >> (threadIdx.x & 48u) & 0xFFFFu) != 0u);
        if (t0 + t < lo || t0 + t >= hi) continue;
        const uint32_t shift = 16u * (t & 1u) + 4u * (t >> 1);
        float y[2] = {y0, y1};
        sc.codes(y);
        w |= static_cast<uint32_t>(y[0]) << shift;
        if (both) w |= static_cast<uint32_t>(y[1]) << (shift + 8u);
        mine |= 0x0F0Fu << shift;
        if (c == 0u)
        {
            sb[t] = static_cast<uint16_t>(sc.scale_bits());
            sb[4u + t] = static_cast<uint16_t>(sc.base_bits());
        }
    }
    *to = mine == 0xFFFFFFFFu ? w : w | (*to & ~mine);
}

// The first waves take values: with a model's format a page's slots of a channel a
// thread, which lie next to each other, in 4 bits the four tokens of two channels that
// share a word.  A word that also holds tokens of before keeps those: each word is
// written by one thread, whatever rows of the call meet in it.  The others take queries
// and keys, 8 channels of a row a thread.  Many short waves: with four rows a wave 2,874
// rows of 32 + 16 heads of 64 take 14.8 us for 12.4, and the values' longer waves at the
// end, behind the others, cost 4.
//   Bound by memory where there are many rows: 2,048 of 32 + 16 heads of 128 (bf16, 51 MB)
// 10.9 us, 4.7 TB/s, a large copy's rate; those 2,874 to 4 bits (32 MB) 11.4, 2.8 TB/s, where
// the vector unit is busy 61% of the CUs' clocks.  One row 3.8 us, 160 rows to 4 bits 4.0: the launch.
template <int XF, int AF, bool I4>
__global__ __launch_bounds__(256) void k_kv_append(AppendParams p)
{
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t id = __builtin_amdgcn_readfirstlane(4u * blockIdx.x + (threadIdx.x >> 6));
    if (id >= p.v_waves)
    {
        const uint32_t row_id = id - p.v_waves, row = row_id / p.row_cols, b = row / p.rows;
        uint32_t u = (row_id - row * p.row_cols) * 64u + lane;
        if (b >= p.batch) return;                         // the last workgroup's waves past the end
        const AppendSeq sq(p, b);
        if (sq.bad && lane == 0u) p.err[ERR_POSITION] = 1u;
        const uint32_t pos = sq.first + (row - b * p.rows);
        if (pos >= sq.end) return;
        if (u < p.q_units)
        {
            const uint32_t d = 8u * u - div_by(u, p.q_per_head) * p.hd;
            store8<AF>(p.q_out, static_cast<uint64_t>(row) * p.heads * p.hd + 8u * u, turn8(p, load8<XF>(p.q, row * p.q_stride + 8u * u), pos, d));
            return;
        }
        u -= p.k_first;                                   // wraps between q_units and k_first
        if (u >= p.k_units) return;
        const int32_t pg = append_page(p, b, pos);
        if (pg < 0) return;
        const uint32_t h = div_by(u, p.per_head), i = u - h * (I4 ? 4u * p.ng : p.hd / 8u), d = 8u * i, slot = pos % OPURE_PAGE_SIZE;
        const bool there = !I4 || d < p.hd;
        f8_t x = {};
        if (there) x = turn8(p, load8<XF>(p.k, row * p.k_stride + h * p.hd + d), pos, d);
        if constexpr (I4) put_k4(p, x, there, static_cast<uint32_t>(pg), h, i, slot);
        else store8<AF>(p.pool, kv_elem(p.layer, p.n_pages, static_cast<uint32_t>(pg), 0u, p.n_kv, h, p.hd, slot, d), x);
        return;
    }
    const uint32_t piece = id / p.v_cols, u = (id - piece * p.v_cols) * 64u + lane, b = piece / p.pieces, i = piece - b * p.pieces;
    const AppendSeq sq(p, b);
    constexpr uint32_t N = I4 ? 4u : OPURE_PAGE_SIZE;     // positions of a piece
    const uint32_t first = (sq.first / N + i) * N, lo = max(first, sq.first), hi = min(first + N, sq.end);
    if (lo >= hi || u >= p.v_units) return;
    const int32_t pg = append_page(p, b, first);
    if (pg < 0) return;
    const uint64_t row0 = static_cast<uint64_t>(b) * p.rows - sq.first;     // a position's row, modulo 2^64
    if constexpr (!I4)
    {
        const uint32_t h = div_by(u, p.v_per_head), d = u - h * p.hd;
        const uint64_t at = kv_elem(p.layer, p.n_pages, static_cast<uint32_t>(pg), 1u, p.n_kv, h, p.hd, 0u, d);
        if (hi - lo == N)
        {
            float x[N];
#pragma unroll
            for (uint32_t t = 0; t < N; ++t) x[t] = load_act<XF>(p.v, (row0 + first + t) * p.v_stride + u);
#pragma unroll
            for (uint32_t t = 0; t < N; t += 8u) store8<AF>(p.pool, at + t, f8_t{x[t], x[t + 1], x[t + 2], x[t + 3], x[t + 4], x[t + 5], x[t + 6], x[t + 7]});
        }
        else
            for (uint32_t t = lo; t < hi; ++t) store_act_rt(p.pool, at + (t - first), load_act<XF>(p.v, (row0 + t) * p.v_stride + u), AF);
    }
    else
    {
        // sixteen lanes a group, channels c and c + 16 of it
        const uint32_t h = div_by(u, p.v_per_head), g = (u - h * 16u * p.ng) >> 4, c = u & 15u, d = 32u * g + c;
        const bool both = d + 16u < p.hd;
        float x[4][2];
#pragma unroll
        for (uint32_t t = 0; t < 4; ++t)
        {
            const uint64_t at = (row0 + min(max(first + t, lo), hi - 1u)) * p.v_stride + h * p.hd + d;
            x[t][0] = load_act<XF>(p.v, at);
            x[t][1] = both ? load_act<XF>(p.v, at + 16u) : x[t][0];
        }
        put_v4(p, x, both, static_cast<uint32_t>(pg), h, g, c, first, lo, hi);
    }
}

uint32_t up_div(uint64_t n, uint64_t d) { return static_cast<uint32_t>((n + d - 1u) / d); }
uint32_t magic(uint32_t d) { return d == 1u ? 0u : static_cast<uint32_t>(((1ull << 32) + d - 1u) / d); }

}  // namespace

using namespace opure_hip;

namespace opure_hip {

uint64_t kv_pool_bytes(const opure_model* m, uint32_t kvfmt, uint32_t n_pages)
{
    const uint64_t planes = static_cast<uint64_t>(m->n_layers) * n_pages * m->n_kv_heads;
    return kvfmt == OPURE_KV_I4 ? planes * BLOCK * groups(m->head_dim) : planes * 2u * OPURE_PAGE_SIZE * m->head_dim * act_bytes(m->afmt);
}

}  // namespace opure_hip

extern "C" int opure_kv_pool_bytes(const opure_model* m, uint32_t kvfmt, uint32_t n_pages, uint64_t* bytes)
{
    OPURE_REQUIRE(m && bytes, OPURE_E_INVALID, "opure_kv_pool_bytes: null argument");
    OPURE_REQUIRE(kvfmt <= OPURE_KV_I4 && m->afmt <= OPURE_A_BF16, OPURE_E_INVALID, "opure_kv_pool_bytes: bad format");
    OPURE_REQUIRE(m->head_dim >= 16 && m->head_dim <= 256 && m->head_dim % 16 == 0, OPURE_E_UNSUPPORTED,
                  "opure_kv_pool_bytes: head_dim %u not in 16..256 step 16", m->head_dim);
    *bytes = kv_pool_bytes(m, kvfmt, n_pages);
    return OPURE_OK;
}

extern "C" int opure_kv_append(opure_dev* dev, const opure_kv_append_args* a)
{
    OPURE_REQUIRE(dev && a && a->model && a->kv && a->kv->pool && a->kv->page_table && a->seq_len && a->k && a->v, OPURE_E_INVALID,
                  "opure_kv_append: null argument");
    const opure_model* m = a->model;
    const opure_kv* kv = a->kv;
    OPURE_REQUIRE(a->kvfmt <= OPURE_KV_I4, OPURE_E_INVALID, "opure_kv_append: bad cache format %u", a->kvfmt);
    OPURE_REQUIRE(m->n_layers >= 1 && m->n_kv_heads >= 1 && m->afmt <= OPURE_A_BF16, OPURE_E_INVALID, "opure_kv_append: bad model");
    OPURE_REQUIRE(a->xfmt == OPURE_A_F32 || a->xfmt == m->afmt, a->xfmt <= OPURE_A_BF16 ? OPURE_E_UNSUPPORTED : OPURE_E_INVALID,
                  "opure_kv_append: rows in format %u for a model in %s: fp32 or the model's", a->xfmt, afmt_name(m->afmt));
    OPURE_REQUIRE(m->head_dim >= 16 && m->head_dim <= 256 && m->head_dim % 16 == 0, OPURE_E_UNSUPPORTED,
                  "opure_kv_append: head_dim %u not in 16..256 step 16", m->head_dim);
    OPURE_REQUIRE(kv->page_size == OPURE_PAGE_SIZE, OPURE_E_UNSUPPORTED, "opure_kv_append: page_size must be %d", OPURE_PAGE_SIZE);
    OPURE_REQUIRE(kv->n_pages >= 1 && kv->max_pages_per_seq >= 1, OPURE_E_INVALID, "opure_kv_append: the cache has no pages");
    OPURE_REQUIRE(a->layer < m->n_layers, OPURE_E_INVALID, "opure_kv_append: layer %u of %u", a->layer, m->n_layers);
    OPURE_REQUIRE(a->batch >= 1 && a->batch <= OPURE_MAX_BATCH_ROWS && a->rows >= 1 && a->rows <= OPURE_MAX_PROMPT_ROWS, OPURE_E_CAPACITY,
                  "opure_kv_append: %u rows x %u sequences outside 1..%d x 1..%d", a->rows, a->batch, OPURE_MAX_PROMPT_ROWS, OPURE_MAX_BATCH_ROWS);
    OPURE_REQUIRE((a->q != nullptr) == (a->q_out != nullptr), OPURE_E_INVALID, "opure_kv_append: q and q_out come together");
    const uint32_t heads = a->q ? m->n_heads : 0u;
    OPURE_REQUIRE(!a->q || heads >= 1, OPURE_E_INVALID, "opure_kv_append: no query heads");
    // the threads' indexes stay in 32 bits, a row's in 24
    OPURE_REQUIRE((static_cast<uint64_t>(heads) + m->n_kv_heads) * a->batch * a->rows <= 1u << 25 &&
                      (static_cast<uint64_t>(heads) + m->n_kv_heads) <= 1u << 15, OPURE_E_CAPACITY,
                  "opure_kv_append: %u x %u rows of %u + %u heads", a->batch, a->rows, heads, m->n_kv_heads);
    const uint64_t slots = static_cast<uint64_t>(kv->max_pages_per_seq) * OPURE_PAGE_SIZE;
    OPURE_REQUIRE(a->max_ctx >= 1 && a->max_ctx <= slots && a->max_ctx <= 0x7FFFFFFFu - OPURE_MAX_PROMPT_ROWS, OPURE_E_CAPACITY,
                  "opure_kv_append: max_ctx %u beyond the page table's %llu", a->max_ctx, (unsigned long long)slots);
    OPURE_REQUIRE(!a->rotate || (m->rope_cos && m->rope_sin && m->rope_max_pos >= a->max_ctx), OPURE_E_INVALID,
                  "opure_kv_append: rotating needs RoPE tables of max_ctx %u positions", a->max_ctx);
    const uint64_t hd = m->head_dim, n = static_cast<uint64_t>(a->batch) * a->rows, xb = act_bytes(a->xfmt), eb = act_bytes(m->afmt);
    OPURE_REQUIRE((!a->q || a->q_stride >= heads * hd) && a->k_stride >= m->n_kv_heads * hd && a->v_stride >= m->n_kv_heads * hd,
                  OPURE_E_INVALID, "opure_kv_append: rows overlap");
    auto address = [](const void* at) { return reinterpret_cast<uintptr_t>(at); };
    OPURE_REQUIRE(((address(a->q) | address(a->k) | address(a->v) | address(a->q_out) | address(kv->pool) | (a->q ? a->q_stride * xb : 0u) |
                    a->k_stride * xb | a->v_stride * xb) & 15u) == 0u, OPURE_E_INVALID,
                  "opure_kv_append: the rows of q, k and v, q_out and pool must be 16-byte aligned");
    OPURE_REQUIRE(!a->rotate || ((address(m->rope_cos) | address(m->rope_sin)) & 15u) == 0u, OPURE_E_INVALID,
                  "opure_kv_append: the RoPE tables must be 16-byte aligned");
    OPURE_REQUIRE(((address(kv->page_table) | address(a->seq_len) | address(a->row_count)) & 3u) == 0u, OPURE_E_INVALID,
                  "opure_kv_append: page_table, seq_len and row_count must be 4-byte aligned");
    // what is written lies apart from everything else, but for queries turned in place
    const uint64_t table = m->rope_max_pos * (hd / 2u) * 4u;
    const struct { const char* name; const void* at; uint64_t bytes; } part[] = {
        {"pool", kv->pool, kv_pool_bytes(m, a->kvfmt, kv->n_pages)},
        {"q_out", a->q_out, n * heads * hd * eb},
        {"q", a->q, ((n - 1u) * a->q_stride + heads * hd) * xb},
        {"k", a->k, ((n - 1u) * a->k_stride + m->n_kv_heads * hd) * xb},
        {"v", a->v, ((n - 1u) * a->v_stride + m->n_kv_heads * hd) * xb},
        {"page_table", kv->page_table, static_cast<uint64_t>(a->batch) * kv->max_pages_per_seq * 4u},
        {"seq_len", a->seq_len, a->batch * 4u},
        {"row_count", a->row_count, a->batch * 4u},
        {"rope_cos", a->rotate ? m->rope_cos : nullptr, table},
        {"rope_sin", a->rotate ? m->rope_sin : nullptr, table}};
    const bool in_place = a->q && a->q == a->q_out && a->xfmt == m->afmt && a->q_stride == heads * hd;
    for (int x = 0; x < 2; ++x)
        for (int y = x + 1; y < 10; ++y)
            OPURE_REQUIRE((x == 1 && y == 2 && in_place) || !overlaps(part[x].at, part[x].bytes, part[y].at, part[y].bytes), OPURE_E_INVALID,
                          "opure_kv_append: %s overlaps %s", part[x].name, part[y].name);
    const DeviceGuard on(dev);
    AppendParams p{};
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.q_out = a->q_out;
    p.pool = kv->pool;
    p.page_table = kv->page_table;
    p.seq_len = a->seq_len;
    p.row_count = a->row_count;
    p.cos = a->rotate ? m->rope_cos : nullptr;
    p.sin = a->rotate ? m->rope_sin : nullptr;
    p.q_stride = a->q_stride;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.heads = heads;
    p.n_kv = m->n_kv_heads;
    p.hd = m->head_dim;
    p.ng = groups(m->head_dim);
    p.rows = a->rows;
    p.n_pages = kv->n_pages;
    p.max_pages = kv->max_pages_per_seq;
    p.layer = a->layer;
    p.cap = a->max_ctx;
    p.err = dev->err;
    const bool i4 = a->kvfmt == OPURE_KV_I4;
    p.q_units = heads * p.hd / 8u;
    p.q_per_head = magic(p.hd / 8u);
    p.k_first = (p.q_units + 3u) & ~3u;
    p.k_units = p.n_kv * (i4 ? 4u * p.ng : p.hd / 8u);
    p.per_head = i4 ? magic(4u * p.ng) : p.q_per_head;
    p.v_units = p.n_kv * (i4 ? 16u * p.ng : p.hd);
    p.v_per_head = magic(i4 ? 16u * p.ng : p.hd);
    p.row_cols = up_div(p.k_first + p.k_units, 64u);
    p.batch = a->batch;
    p.v_cols = up_div(p.v_units, 64u);
    p.pieces = i4 ? (a->rows + 2u) / 4u + 1u : (a->rows + 14u) / 16u + 1u;
    const uint64_t v_waves = static_cast<uint64_t>(a->batch) * p.pieces * p.v_cols, waves = v_waves + static_cast<uint64_t>(a->batch) * a->rows * p.row_cols;
    OPURE_REQUIRE(waves < 1u << 26, OPURE_E_CAPACITY, "opure_kv_append: too many workgroups");
    p.v_waves = static_cast<uint32_t>(v_waves);
    auto go = [&](auto xf, auto af) {
        constexpr int XF = decltype(xf)::value, AF = decltype(af)::value;
        const dim3 grid(up_div(waves, 4u)), block(256);
        if (i4) OPURE_LAUNCH(dev, (k_kv_append<XF, AF, true>), grid, block, 0, p);
        else OPURE_LAUNCH(dev, (k_kv_append<XF, AF, false>), grid, block, 0, p);
    };
    typedef std::integral_constant<int, OPURE_A_F32> F32;
    typedef std::integral_constant<int, OPURE_A_F16> F16;
    typedef std::integral_constant<int, OPURE_A_BF16> BF16;
    if (m->afmt == OPURE_A_F32) go(F32{}, F32{});
    else if (m->afmt == OPURE_A_F16) a->xfmt == OPURE_A_F32 ? go(F32{}, F16{}) : go(F16{}, F16{});
    else a->xfmt == OPURE_A_F32 ? go(F32{}, BF16{}) : go(BF16{}, BF16{});
    OPURE_LAUNCH_CHECK("k_kv_append");
    return OPURE_OK;
}
