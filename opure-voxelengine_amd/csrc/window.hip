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

using namespace opure_dev_math;

namespace {

struct WinParams {
    const void* q;
    void* out;
    const void* pool;
    const int32_t* page_table;
    const int32_t* seq_len;
    float* ml;           // [batch * rows * n_heads][2]: each query row's maximum and sum
    float* weights;
    uint64_t weights_batch_stride;
    uint32_t weights_stride;
    uint32_t n_heads, n_kv, hd, rows, n_pages, max_pages, layer, afmt;
    uint32_t window, sinks;       // window >= 1: 2^31 - 1 sees everything
    uint32_t cap;                 // positions that may be read: min(max_ctx, the table's)
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

__global__ __launch_bounds__(64) void k_win_row(WinParams p)
{
    __shared__ float qs[256];
    const uint32_t head = blockIdx.x % p.n_heads, row = blockIdx.x / p.n_heads;
    const uint32_t b = row / p.rows, j = row - b * p.rows, kh = head / (p.n_heads / p.n_kv), lane = threadIdx.x;
    const WinSeq sq = win_seq(p, p.seq_len[b]);
    const uint64_t at = (static_cast<uint64_t>(row) * p.n_heads + head) * p.hd;
    for (uint32_t d = lane; d < p.hd; d += 64u) qs[d] = load_act_rt(p.q, at + d, p.afmt);
    __syncthreads();
    float m, l, o[4];
    win_row(p, qs, b, kh, sq.ctx + j, sq.total, m, l, o);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64u * i < p.hd) store_act_rt(p.out, at + lane + 64u * i, l == 0.0f ? 0.0f : __fdiv_rn(o[i], l), p.afmt);
    if (lane == 0u && p.ml)
    {
        p.ml[2ull * blockIdx.x] = m;
        p.ml[2ull * blockIdx.x + 1u] = l;
    }
}

// The weights of 64 positions of a (sequence, KV head): a lane a position, the
// rows that see it and their heads in order.
__global__ __launch_bounds__(64) void k_win_weights(WinParams p)
{
    const uint32_t kh = blockIdx.y, b = blockIdx.z, t = blockIdx.x * 64u + threadIdx.x;
    const uint32_t G = p.n_heads / p.n_kv, hd = p.hd;
    const WinSeq sq = win_seq(p, p.seq_len[b]);
    if (t >= sq.total) return;
    const int32_t pg = win_page(p, p.page_table + static_cast<uint64_t>(b) * p.max_pages, t);
    const uint64_t kat = kv_elem(p.layer, p.n_pages, pg >= 0 ? static_cast<uint32_t>(pg) : 0u, 0u, p.n_kv, kh, hd, t % OPURE_PAGE_SIZE, 0u);
    float sum = 0.0f;
    bool any = false;
    for (uint32_t j = 0; j < p.rows; ++j)
    {
        if (!win_sees(p, sq.ctx + j, t)) continue;
        any = true;
        for (uint32_t g = 0; g < G; ++g)
        {
            const uint64_t row = (static_cast<uint64_t>(b) * p.rows + j) * p.n_heads + kh * G + g;
            float s = __builtin_nanf("");
            if (pg >= 0)
            {
                float acc = 0.0f;
                for (uint32_t d = 0; d < hd; ++d)
                    acc = __fmaf_rn(load_act_rt(p.q, row * hd + d, p.afmt), load_act_rt(p.pool, kat + d, p.afmt), acc);
                s = __fmul_rn(acc, p.scale);
            }
            const float m = p.ml[2u * row], l = p.ml[2u * row + 1u], ms = m == -__builtin_huge_valf() ? 0.0f : m;
            sum += l == 0.0f ? 0.0f : __fdiv_rn(expf_ref(__fsub_rn(s, ms)), l);
        }
    }
    if (any) p.weights[b * p.weights_batch_stride + static_cast<uint64_t>(kh) * p.weights_stride + t] += sum;
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
    // a query row's index in its sequence and KV head stays in 32 bits, and the head grids in theirs
    OPURE_REQUIRE(m->n_heads <= 65535u, OPURE_E_CAPACITY, "window attention: %u heads", m->n_heads);
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

uint64_t win_ws_bytes(const opure_attn_window_args* a)
{
    return a->weights ? static_cast<uint64_t>(a->batch) * a->rows * a->model->n_heads * 8u : 0u;
}

}  // namespace

using namespace opure_hip;

extern "C" int opure_attn_window_reserve(opure_dev* dev, const opure_attn_window_args* a)
{
    OPURE_REQUIRE(dev, OPURE_E_INVALID, "opure_attn_window_reserve: null device");
    const int rc = win_validate(a);
    if (rc) return rc;
    const DeviceGuard on(dev);
    return ensure_workspace(dev, win_ws_bytes(a));
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
    rc = ensure_workspace(dev, win_ws_bytes(a));
    if (rc) return rc;
    WinParams p{};
    p.q = a->q;
    p.out = a->out;
    p.pool = a->kv->pool;
    p.page_table = a->kv->page_table;
    p.seq_len = a->seq_len;
    p.ml = a->weights ? static_cast<float*>(dev->ws) : nullptr;
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
    OPURE_LAUNCH(dev, k_win_row, dim3(a->batch * a->rows * p.n_heads), dim3(64), 0, p);
    OPURE_LAUNCH_CHECK("k_win_row");
    if (p.weights)
    {
        OPURE_LAUNCH(dev, k_win_weights, dim3((a->max_ctx + 63u) / 64u, p.n_kv, a->batch), dim3(64), 0, p);
        OPURE_LAUNCH_CHECK("k_win_weights");
    }
    return OPURE_OK;
}
