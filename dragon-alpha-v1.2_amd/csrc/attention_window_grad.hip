// The gradient of windowed attention (attention_window.hip has the definition).  With P = exp(scale * S - lse) on the pairs
// that see each other, D[i] = <dY[i], Y[i]> and dS = P * (dY.V^T - D):
//     dQ = scale * dS.K      dK = scale * dS^T.Q      dV = P^T.dY        (dK and dV over all query heads that share the head)
// P is computed again from Q, K and lse, never stored.  Two kernels, so that every sum has one owner and no result depends on
// the order of arrival: window_grad_q owns 128 queries and walks over the keys they see, window_grad_kv owns 128 keys and
// walks over the queries that see them, head by head of the group.  That is seven products of which five are necessary:
// the score and the dY.V^T products happen in both.  Bound by the FP32 matrix pipe.
//
// A key tile with sinks is seen by all queries behind it, any other by window + 128 of them: the sinks' tile is cut along the
// queries (as every tile is where there are few), each part leaves its sums in the caller's buffer and
// window_grad_join adds them in order.
#include "token_mixer.h"
#include "attention_window.h"
#include "runtime_internal.h"
#include "../../include/dragon_hip_gemm.h"

namespace dragon {
bool window_arguments_ok(int N, int head, int kv_head, int QL, int VL, int dk4, int dv4, int window, int sinks);
namespace {

constexpr int GQ = 128;    // queries per workgroup of window_grad_q
constexpr int GK = 128;    // keys per workgroup of window_grad_kv

struct WindowGrad {
    WindowParams w;          // Y, Lse: what the forward pass left
    const float* dY; float* dQ; float* dK; float* dV;
    float* D;                // [N, head, QL]
    float scale;
    int ktiles, sink_tiles, sink_parts, parts;
    float* sink_sums; float* sums;     // [N, kv_head, keys][parts][dk4 + dv4]
};

// ---------------------------------------------------------------- D[i] = <dY[i], Y[i]>
__global__ __launch_bounds__(NTHREADS) void window_delta(const WindowGrad p) {
    const long long row = (long long)blockIdx.x * (NTHREADS / 32) + (threadIdx.x >> 5);
    if (row >= (long long)p.w.N * p.w.head * p.w.QL) return;
    const long long nh = row / p.w.QL;
    const int n = (int)(nh / p.w.head), hd = (int)(nh - (long long)n * p.w.head), i = (int)(row - nh * p.w.QL);
    const int d = 4 * (threadIdx.x & 31);
    float sum = 0.0f;
    const int ql = p.w.QLens ? min(p.w.QLens[n], p.w.QL) : p.w.QL;
    if (i < ql && d < p.w.dv4) {
        const size_t at = n * p.w.y.n + hd * p.w.y.h + (size_t)i * p.w.y.l + d;
        const v4f a = *(const v4f*)(p.dY + at), b = *(const v4f*)(p.w.Y + at);
        sum = (a.x * b.x + a.y * b.y) + (a.z * b.z + a.w * b.w);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
    if ((threadIdx.x & 31) == 0) p.D[row] = sum;
}

// ---------------------------------------------------------------- dQ
template <int DB, int DC>
__global__ __launch_bounds__(NTHREADS, 2) void window_grad_q(const WindowGrad a) {
    constexpr int DW = DB * 32, NG = DC * 4;
    const WindowParams& p = a.w;
    __shared__ __attribute__((aligned(16))) float Ks[2][32 * DW];
    __shared__ __attribute__((aligned(16))) float Vs[2][32 * DW];
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const WindowJob job = window_job(p, blockIdx.x);
    const WindowLens len = window_lens(p, job.n);
    const int q0 = job.qt * GQ, i = q0 + wave * 32 + r;
    const size_t stat = ((size_t)job.n * p.head + job.hd) * p.QL + min(i, p.QL - 1);
    const int qn = min(q0 + GQ, len.ql), off = len.vl - len.ql;
    const WindowRange range = window_range(p, q0 + off, qn - 1 + off, q0 < qn, len.vl);
    const int nsink = (range.sink_end + 31) / 32, steps = nsink + (max(range.hi - range.low, 0) + 31) / 32;
    const bool live = i < len.ql;
    const int pos = live ? i + off : -1;
    const int w0 = q0 + wave * 32 + off, w1 = min(q0 + wave * 32 + 32, len.ql) - 1 + off;

    v4f qf[NG], gf[NG];
    mix_load_cols<NG>(qf, p.Q + job.n * p.q.n + job.hd * p.q.h + (size_t)min(i, p.QL - 1) * p.q.l, live, p.dk4, h);
    mix_load_cols<NG>(gf, a.dY + job.n * p.y.n + job.hd * p.y.h + (size_t)min(i, p.QL - 1) * p.y.l, live, p.dv4, h);
#pragma unroll
    for (int g = 0; g < NG; g++) qf[g] *= p.c;
    const float lse = live ? p.Lse[stat] * MIX_LOG2E : 0.0f, D = live ? a.D[stat] : 0.0f;
    const v16f from = (v16f)(-lse);                         // where the score products start: P = exp2 of the result

    const float* Kb = p.K + job.n * p.k.n + job.kvh * p.k.h;
    const float* Vb = p.V + job.n * p.v.n + job.kvh * p.v.h;
    MixTile<DW, 32, true> kt, vt;
    MixColumns<DW, true> cols;
    cols.init(r, h);
    kt.init(t, p.k.l, p.dk4);
    vt.init(t, p.v.l, p.dv4);
    auto key_of = [&](int s) { return s < nsink ? s * 32 : range.low + (s - nsink) * 32; };
    const unsigned klds = mix_lds(Ks[0]) + wave * 1024, vlds = mix_lds(Vs[0]) + wave * 1024;
    auto fetch = [&](int s, int into) {
        const int key0 = key_of(s), left = (s < nsink ? range.sink_end : range.hi) - key0;
        kt.fetch(Kb + (size_t)key0 * p.k.l, left, p.k.l, klds + into * (32 * DW * 4));
        vt.fetch(Vb + (size_t)key0 * p.v.l, left, p.v.l, vlds + into * (32 * DW * 4));
    };
    v16f o[DC];
#pragma unroll
    for (int b = 0; b < DC; b++) o[b] = (v16f)(0.0f);
    if (steps > 0) fetch(0, 0);
    mix_wait();
    __syncthreads();
    auto step = [&](auto bufc, int s) {
        constexpr int buf = decltype(bufc)::value;
        if (s + 1 < steps) fetch(s + 1, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        const int key0 = key_of(s), limit = s < nsink ? range.sink_end : range.hi, end = min(key0 + 32, limit);
        const bool sees = w0 <= w1 && (s < nsink || (key0 <= w1 && (end - 1 > w0 - p.window || key0 < p.sinks)));
        if (sees) {
            v16f sc = from, dp = (v16f)(0.0f);
            mix_rows_product<DW, NG>(sc, Ks[buf], qf, r, h);
            mix_rows_product<DW, NG>(dp, Vs[buf], gf, r, h);
#pragma unroll
            for (int v = 0; v < 16; v++) sc[v] = __builtin_amdgcn_exp2f(sc[v]) * (dp[v] - D);
            // keys behind a query (or behind the last key), and before its window: tested only where some query has them
            if (key0 + 31 > w0 || key0 + 32 > limit || q0 + wave * 32 + 32 > len.ql) {
                const int top = min(pos, limit - 1) - key0 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (mix_row(v, 0) > top) sc[v] = 0.0f;
            }
            if (s >= nsink && key0 <= w1 - p.window) {
                const int low = pos - p.window - key0 - 4 * h, sink = p.sinks - key0 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (mix_row(v, 0) <= low && mix_row(v, 0) >= sink) sc[v] = 0.0f;
            }
            mix_columns_product<DW, DC, true>(o, Ks[buf], sc, cols, r, h);
        }
        mix_wait();
        __syncthreads();
    };
    for (int s = 0; s < steps; s += 2) {
        step(std::integral_constant<int, 0>{}, s);
        if (s + 1 < steps) step(std::integral_constant<int, 1>{}, s + 1);
    }
    if (i < p.QL) mix_store_row<DC>(a.dQ + job.n * p.q.n + job.hd * p.q.h + (size_t)i * p.q.l, o, a.scale, p.dk4, h);
}

// ---------------------------------------------------------------- dK, dV
template <int DB, int DC>
__global__ __launch_bounds__(NTHREADS, DB > 2 ? 1 : 2) void window_grad_kv(const WindowGrad a) {
    constexpr int DW = DB * 32, NG = DC * 4;
    const WindowParams& p = a.w;
    __shared__ __attribute__((aligned(16))) float Qs[2][32 * DW];
    __shared__ __attribute__((aligned(16))) float Gs[2][32 * DW];
    __shared__ __attribute__((aligned(16))) float Ls[2][32], Ds[2][32];
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;

    // key tiles in order (the first are seen by the most queries), the sinks' in sink_parts each
    const int nkv = p.N * p.kv_head, group = p.head / p.kv_head;
    const int x = mix_uniform(blockIdx.x / nkv), kv = blockIdx.x - x * nkv;
    const bool sink_tile = x < a.sink_tiles * a.sink_parts;
    const int parts = sink_tile ? a.sink_parts : a.parts;
    const int y = sink_tile ? x : x - a.sink_tiles * a.sink_parts;
    const int tile = mix_uniform(y / parts), part = y - tile * parts;
    const int n = mix_uniform(kv / p.kv_head), kvh = kv - n * p.kv_head;
    const int k0 = (sink_tile ? tile : a.sink_tiles + tile) * GK;
    const WindowLens len = window_lens(p, n);
    const int off = len.vl - len.ql;
    const int key = k0 + wave * 32 + r, k1 = min(k0 + GK, len.vl);
    const bool live = key < len.vl;
    const int u0 = k0 + wave * 32, u1 = min(u0 + 32, len.vl) - 1;      // the wavefront's keys

    // the queries that see a key of the tile: [lo, hi)
    const int lo = max(k0 - off, 0);
    const int hi = k0 < k1 ? (k0 < p.sinks ? len.ql : min(len.ql, k1 - 1 + p.window - off)) : 0;
    const int per_head = (max(hi - lo, 0) + 31) / 32, total = per_head * group;
    const int first = mix_uniform((int)((long long)total * part / parts)), last = mix_uniform((int)((long long)total * (part + 1) / parts));

    v4f kf[NG], vf[NG];
    mix_load_cols<NG>(kf, p.K + n * p.k.n + kvh * p.k.h + (size_t)min(key, p.VL - 1) * p.k.l, live, p.dk4, h);
    mix_load_cols<NG>(vf, p.V + n * p.v.n + kvh * p.v.h + (size_t)min(key, p.VL - 1) * p.v.l, live, p.dv4, h);
#pragma unroll
    for (int g = 0; g < NG; g++) kf[g] *= p.c;

    MixTile<DW, 32, true> qt, gt;
    MixColumns<DW, true> cols;
    cols.init(r, h);
    qt.init(t, p.q.l, p.dk4);
    gt.init(t, p.y.l, p.dv4);
    float stat_reg = 0.0f;
    const unsigned qlds = mix_lds(Qs[0]) + wave * 1024, glds = mix_lds(Gs[0]) + wave * 1024;
    // the step after (head g0 of the group, query tile i0) is (g0, i0 + 32) or the next head's first
    auto fetch = [&](int g, int i0, int into) {
        const int hd = kvh * group + g;
        qt.fetch(p.Q + n * p.q.n + hd * p.q.h + (size_t)i0 * p.q.l, hi - i0, p.q.l, qlds + into * (32 * DW * 4));
        gt.fetch(a.dY + n * p.y.n + hd * p.y.h + (size_t)i0 * p.y.l, hi - i0, p.y.l, glds + into * (32 * DW * 4));
        const size_t row = ((size_t)n * p.head + hd) * p.QL + i0 + (t & 31);
        if (t < 64) stat_reg = i0 + (t & 31) < hi ? (t < 32 ? p.Lse[row] * MIX_LOG2E : a.D[row]) : 0.0f;
    };
    auto store = [&](int into) {
        if (t < 32) Ls[into][t] = stat_reg;
        else if (t < 64) Ds[into][t - 32] = stat_reg;
    };
    v16f dk[DC], dv[DC];
#pragma unroll
    for (int b = 0; b < DC; b++) { dk[b] = (v16f)(0.0f); dv[b] = (v16f)(0.0f); }
    int g = 0, i0 = lo;
    if (first < last) {
        g = mix_uniform(first / per_head);
        i0 = lo + (first - g * per_head) * 32;
        fetch(g, i0, 0);
    }
    mix_wait();
    store(0);
    __syncthreads();
    auto step = [&](auto bufc, int s) {
        constexpr int buf = decltype(bufc)::value;
        const bool more = s + 1 < last;
        const bool turn = i0 + 32 >= hi;
        const int next_g = turn ? g + 1 : g, next_i0 = turn ? lo : i0 + 32;
        if (more) fetch(next_g, next_i0, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        const int p0 = i0 + off, p1 = min(i0 + 32, hi) - 1 + off;      // the step's positions
        const bool sees = u0 <= u1 && p1 >= u0 && (p0 < u1 + p.window || u0 < p.sinks);
        if (sees) {
            v16f sc = (v16f)(0.0f), dp = (v16f)(0.0f);
            mix_rows_product<DW, NG>(sc, Qs[buf], kf, r, h);
            mix_rows_product<DW, NG>(dp, Gs[buf], vf, r, h);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const v4f lse = *(const v4f*)&Ls[buf][8 * q + 4 * h], D = *(const v4f*)&Ds[buf][8 * q + 4 * h];
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    sc[4 * q + w] = __builtin_amdgcn_exp2f(sc[4 * q + w] - lse[w]);
                    dp[4 * q + w] = dp[4 * q + w] - D[w];
                }
            }
            // queries before a key, those whose window has passed it, and rows behind the last: tested only where there are any.
            // Both factors are cleared: dP may be anything where nothing is seen.
            if (p0 < u1 || i0 + 32 > hi || u0 + 32 > len.vl) {
                const int low = (live ? key : 0x3fffffff) - p0 - 4 * h, top = hi - 1 - i0 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (mix_row(v, 0) < low || mix_row(v, 0) > top) sc[v] = dp[v] = 0.0f;
            }
            if (p1 >= u0 + p.window) {
                const int top = key < p.sinks ? 0x3fffffff : key + p.window - 1 - p0 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (mix_row(v, 0) > top) sc[v] = dp[v] = 0.0f;
            }
#pragma unroll
            for (int v = 0; v < 16; v++) dp[v] *= sc[v];
            mix_columns_product<DW, DC, true>(dv, Gs[buf], sc, cols, r, h);
            mix_columns_product<DW, DC, true>(dk, Qs[buf], dp, cols, r, h);
        }
        mix_wait();
        if (more) store(buf ^ 1);
        __syncthreads();
        g = next_g;
        i0 = next_i0;
    };
    for (int s = first; s < last; s += 2) {
        step(std::integral_constant<int, 0>{}, s);
        if (s + 1 < last) step(std::integral_constant<int, 1>{}, s + 1);
    }
    if (key >= p.VL) return;
    if (parts == 1) {
        mix_store_row<DC>(a.dK + n * p.k.n + kvh * p.k.h + (size_t)key * p.k.l, dk, a.scale, p.dk4, h);
        mix_store_row<DC>(a.dV + n * p.v.n + kvh * p.v.h + (size_t)key * p.v.l, dv, 1.0f, p.dv4, h);
    } else {
        const int sink_rows = a.sink_tiles * GK;
        const size_t row = sink_tile ? (size_t)kv * sink_rows + key : (size_t)kv * (p.VL - sink_rows) + key - sink_rows;
        float* at = (sink_tile ? a.sink_sums : a.sums) + (row * parts + part) * (p.dk4 + p.dv4);
        mix_store_row<DC>(at, dk, a.scale, p.dk4, h);
        mix_store_row<DC>(at + p.dk4, dv, 1.0f, p.dv4, h);
    }
}

// the parts of the keys [key0, key0 + rows) of every key / value head, in order
__global__ __launch_bounds__(NTHREADS) void window_grad_join(const WindowGrad a, const float* sums, int key0, int rows, int stride, int parts) {
    const WindowParams& p = a.w;
    const int width = p.dk4 + p.dv4, per = width / 4;
    const long long x = (long long)blockIdx.x * NTHREADS + threadIdx.x;
    const long long row = x / per;
    if (row >= (long long)p.N * p.kv_head * rows) return;
    const int d = 4 * (int)(x - row * per);
    const int kv = (int)(row / rows), key = (int)(row - (long long)kv * rows);
    const float* at = sums + ((size_t)kv * stride + key) * parts * width + d;
    v4f s = *(const v4f*)at;
    for (int k = 1; k < parts; k++) s += *(const v4f*)(at + (size_t)k * width);
    const int n = kv / p.kv_head, kvh = kv - n * p.kv_head;
    if (d < p.dk4) *(v4f*)(a.dK + n * p.k.n + kvh * p.k.h + (size_t)(key0 + key) * p.k.l + d) = s;
    else *(v4f*)(a.dV + n * p.v.n + kvh * p.v.h + (size_t)(key0 + key) * p.v.l + d - p.dk4) = s;
}

// ---------------------------------------------------------------- host side
struct WindowGradPlan { int ktiles, sink_tiles, sink_parts, parts; };

WindowGradPlan window_grad_plan(int N, int head, int kv_head, int QL, int VL, int window, int sinks) {
    WindowGradPlan x;
    const long long group = head / kv_head;
    x.ktiles = (VL + GK - 1) / GK;
    const long long all = ((QL + 31LL) / 32) * group;          // steps of a tile that every query sees
    const long long reach = window == 0 || window >= VL ? QL : (long long)window + GK < QL ? window + GK : QL;
    const long long steps = ((reach + 31) / 32) * group;
    const long long base = (long long)N * kv_head * x.ktiles;
    long long parts = base >= 256 ? 1 : (512 + base - 1) / base;
    if (parts > steps / 8) parts = steps / 8;
    x.parts = (int)(parts < 1 ? 1 : parts > 16 ? 16 : parts);
    x.sink_tiles = x.sink_parts = 0;
    if (window != 0 && window < VL && sinks > 0) {
        const long long least = steps / x.parts > 8 ? steps / x.parts : 8;
        const long long sp = (all + least - 1) / least;
        x.sink_parts = (int)(sp < 1 ? 1 : sp > 64 ? 64 : sp);
        if (x.sink_parts > x.parts) x.sink_tiles = (int)(((long long)(sinks < VL ? sinks : VL) + GK - 1) / GK);
        if (x.sink_tiles > x.ktiles) x.sink_tiles = x.ktiles;
        if (x.sink_tiles == 0) x.sink_parts = 0;
    }
    return x;
}

// floats of D, of the sinks' tiles' parts, of the others'
struct WindowGradBuffer { long long d, sink, rest; };
WindowGradBuffer window_grad_buffer(const WindowGradPlan& x, int N, int head, int kv_head, int QL, int VL, int width) {
    WindowGradBuffer b;
    const long long sink_rows = (long long)x.sink_tiles * GK < VL ? (long long)x.sink_tiles * GK : VL;
    b.d = ((long long)N * head * QL + 3) / 4 * 4;
    b.sink = x.sink_tiles > 0 ? (long long)N * kv_head * x.sink_tiles * GK * x.sink_parts * width : 0;
    b.rest = x.parts > 1 ? (long long)N * kv_head * (VL - sink_rows) * x.parts * width : 0;
    return b;
}

}  // namespace
}  // namespace dragon

using namespace dragon;

extern "C" {

int64_t dragon_Cuda_attention_window_backward_bufsize(int32_t N, int32_t head, int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4,
                                                      int32_t dV4, int32_t window, int32_t sinks) {
    if (!window_arguments_ok(N, head, kv_head, QL, VL, dK4, dV4, window, sinks)) return -1;
    const WindowGradBuffer b = window_grad_buffer(window_grad_plan(N, head, kv_head, QL, VL, window, sinks), N, head, kv_head, QL, VL, dK4 + dV4);
    return (b.d + b.sink + b.rest) * 4;
}

int dragon_Cuda_attention_window_backward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV, int64_t dY,
                                          int64_t dLse, int64_t dDeltaY, int64_t dDeltaQ, int64_t dDeltaK, int64_t dDeltaV,
                                          int64_t dQLens, int64_t dVLens, int64_t dBuf, int64_t buf_size, int32_t N, int32_t head,
                                          int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4, int32_t dV4, int32_t head_inner,
                                          float scale, int32_t window, int32_t sinks) {
    if (streams == nullptr || length < 1 || length > 10) return hipErrorInvalidValue;
    if (dQ == 0 || dK == 0 || dV == 0 || dY == 0 || dLse == 0 || dDeltaY == 0 || dDeltaQ == 0 || dDeltaK == 0 || dDeltaV == 0 ||
        !mix_aligned16(dQ) || !mix_aligned16(dK) || !mix_aligned16(dV) || !mix_aligned16(dY) || !mix_aligned16(dDeltaY) ||
        !mix_aligned16(dDeltaQ) || !mix_aligned16(dDeltaK) || !mix_aligned16(dDeltaV) || (dLse & 3) || (dQLens & 3) || (dVLens & 3))
        return hipErrorInvalidValue;
    if (!window_arguments_ok(N, head, kv_head, QL, VL, dK4, dV4, window, sinks) || !(scale - scale == 0.0f))
        return hipErrorInvalidValue;
    const WindowGradPlan plan = window_grad_plan(N, head, kv_head, QL, VL, window, sinks);
    const WindowGradBuffer b = window_grad_buffer(plan, N, head, kv_head, QL, VL, dK4 + dV4);
    const long long need = (b.d + b.sink + b.rest) * 4;
    if (dBuf == 0 || !mix_aligned16(dBuf) || buf_size < need) return hipErrorInvalidValue;

    WindowGrad a;
    WindowParams& p = a.w;
    p.Q = (const float*)(intptr_t)dQ; p.K = (const float*)(intptr_t)dK; p.V = (const float*)(intptr_t)dV;
    p.Y = (float*)(intptr_t)dY; p.Lse = (float*)(intptr_t)dLse;
    p.QLens = (const int*)(intptr_t)dQLens; p.VLens = (const int*)(intptr_t)dVLens;
    p.N = N; p.head = head; p.kv_head = kv_head; p.QL = QL; p.VL = VL; p.dk4 = dK4; p.dv4 = dV4;
    p.q = mix_layout(head_inner, head, QL, dK4); p.y = mix_layout(head_inner, head, QL, dV4);
    p.k = mix_layout(head_inner, kv_head, VL, dK4); p.v = mix_layout(head_inner, kv_head, VL, dV4);
    p.window = window == 0 || window > QL + VL ? QL + VL : window;
    p.sinks = sinks;
    p.c = scale * MIX_LOG2E;
    p.qtiles = (QL + GQ - 1) / GQ; p.parts = 1; p.part = nullptr;
    a.dY = (const float*)(intptr_t)dDeltaY;
    a.dQ = (float*)(intptr_t)dDeltaQ; a.dK = (float*)(intptr_t)dDeltaK; a.dV = (float*)(intptr_t)dDeltaV;
    a.D = (float*)(intptr_t)dBuf;
    a.scale = scale;
    a.ktiles = plan.ktiles; a.sink_tiles = plan.sink_tiles; a.sink_parts = plan.sink_parts; a.parts = plan.parts;
    a.sink_sums = a.D + b.d; a.sums = a.sink_sums + b.sink;
    split_ledger_touch(a.dQ, (size_t)N * head * QL * dK4 * 4);
    split_ledger_touch(a.dK, (size_t)N * kv_head * VL * dK4 * 4);
    split_ledger_touch(a.dV, (size_t)N * kv_head * VL * dV4 * 4);
    split_ledger_touch(a.D, (size_t)need);

    hipStream_t s = (hipStream_t)(intptr_t)streams[0];
    const dim3 block(NTHREADS);
    const long long rows = (long long)N * head * QL;
    hipLaunchKernelGGL(window_delta, dim3((unsigned)((rows + NTHREADS / 32 - 1) / (NTHREADS / 32))), block, 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 gq((unsigned)((long long)N * head * p.qtiles));
    const dim3 gk((unsigned)((long long)N * kv_head * (plan.sink_tiles * plan.sink_parts + (plan.ktiles - plan.sink_tiles) * plan.parts)));
    const int dmax = dK4 > dV4 ? dK4 : dV4;
#define GRAD_CASE(DB_, DC_)                                                           \
    do {                                                                              \
        hipLaunchKernelGGL((window_grad_kv<DB_, DC_>), gk, block, 0, s, a);           \
        e = hipGetLastError();                                                        \
        if (e != hipSuccess) return e;                                                \
        hipLaunchKernelGGL((window_grad_q<DB_, DC_>), gq, block, 0, s, a);            \
        e = hipGetLastError();                                                        \
        if (e != hipSuccess) return e;                                                \
    } while (0)
    switch ((dmax + 31) / 32) {
        case 1: GRAD_CASE(1, 1); break;
        case 2: GRAD_CASE(2, 2); break;
        case 3: GRAD_CASE(4, 3); break;
        default: GRAD_CASE(4, 4); break;
    }
#undef GRAD_CASE
    const int sink_rows = plan.sink_tiles * GK < VL ? plan.sink_tiles * GK : VL;
    auto join = [&](const float* sums, int key0, int n_rows, int stride, int parts) {
        const long long items = (long long)N * kv_head * n_rows * ((dK4 + dV4) / 4);
        hipLaunchKernelGGL(window_grad_join, dim3((unsigned)((items + NTHREADS - 1) / NTHREADS)), block, 0, s, a, sums, key0, n_rows, stride, parts);
        return hipGetLastError();
    };
    if (plan.sink_tiles > 0) e = join(a.sink_sums, 0, sink_rows, plan.sink_tiles * GK, plan.sink_parts);
    if (e == hipSuccess && plan.parts > 1 && VL > sink_rows) e = join(a.sums, sink_rows, VL - sink_rows, VL - sink_rows, plan.parts);
    return e;
}

}  // extern "C"
