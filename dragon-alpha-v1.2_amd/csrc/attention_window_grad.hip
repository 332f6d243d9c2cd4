// The gradient of windowed attention (attention_window.hip has the definition).  With P = exp(scale * S - lse) on the pairs
// that see each other, D[i] = <dY[i], Y[i]> and dS = P * (dY.V^T - D):
//     dQ = scale * dS.K      dK = scale * dS^T.Q      dV = P^T.dY        (dK and dV over all query heads that share the head)
// P is computed again from Q, K and lse, never stored.  Two kernels, so that every sum has one owner and no result depends on
// the order of arrival: window_grad_q owns 128 (query, head) rows and walks over the keys they see, window_grad_kv owns 128 keys and
// walks over the queries that see them, head by head of the group.  That is seven products of which five are necessary:
// the score and the dY.V^T products happen in both.  Bound by the FP32 matrix pipe: 32 heads of 128 on 8 of keys and values,
// 8192 queries under a window of 1024 take 1.72 ms in window_grad_q and 2.26 in window_grad_kv, 113 TFLOP/s in either and the
// pipes busy for three quarters of the time.
//
// Both run eight wavefronts, two per 32 queries (or keys) and on one SIMD.  The first forms S and P, hands P over through LDS
// and, in window_grad_kv, adds up dV = P^T.dY; the second forms dY.V^T, takes P and adds up dK = dS^T.Q or dQ = dS.K.  Each
// then keeps one operand and one accumulator in registers instead of two.  (One wavefront for everything took 512 registers,
// ran alone on its SIMD and left the matrix pipe idle for half of the time: dK and dV at 32 x 8192 x 128 under a window of
// 1024 in 3.3 ms.)  One barrier a step, between the products: behind it P is there, the next step's tiles have landed, and
// those of the step before are free, so three buffers.
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
    float* stats;            // [2][N, head, QL]: lse and D, zeros behind the queries
    long long rows;          // N * head * QL
    float scale;
    int ktiles, workers;     // key tiles of a key / value head; workgroups of window_grad_kv
    int snap;                // steps that a cut through a tile costs (two beginnings and ends, a piece written and read)
    long long* before;       // [N * ktiles + 1]: the steps of all key tiles before this one, of one key / value head; then the most of a tile
    float* pieces;           // [2 * workers][128][dk4 + dv4]
    int2* cut;               // [N * ktiles, kv_head]: the workers of a tile's first and last piece
    int sink_blocks;         // 16 keys each; 0: the sinks' tiles walk over all queries like the others
    int sink_parts;          // SINK_QUERIES queries each
    float* sinks;            // [N, kv_head][sink_blocks][sink_parts][16][dk4 + dv4]
};

// ---------------------------------------------------------------- the rows' statistics, and the work to deal
// the queries that see a key of tile `tile`: [lo, hi)
struct WindowQueries { int lo, hi; };
__device__ __forceinline__ WindowQueries window_queries(const WindowGrad& a, int tile, WindowLens len) {
    const WindowParams& p = a.w;
    const int k0 = tile * GK, k1 = min(k0 + GK, len.vl), off = len.vl - len.ql;
    WindowQueries x;
    x.lo = max(k0 - off, 0);
    x.hi = k0 < k1 ? (k0 < p.sinks && a.sink_blocks == 0 ? len.ql : min(len.ql, k1 - 1 + p.window - off)) : 0;
    return x;
}
// steps of `per` queries of one query head
__device__ __forceinline__ int window_steps(WindowQueries x, int per) { return (max(x.hi - x.lo, 0) + per - 1) / per; }

__global__ __launch_bounds__(NTHREADS) void window_delta(const WindowGrad a) {
    const WindowParams& p = a.w;
    if (blockIdx.x == gridDim.x - 1) {   // the running sum of the tiles' steps, and the most of one
        __shared__ long long sum[NTHREADS];
        const int t = threadIdx.x, group = p.head / p.kv_head;
        const long long tiles = (long long)p.N * a.ktiles;
        long long base = 0, most = 0;
        for (long long x0 = 0; x0 < tiles; x0 += NTHREADS) {
            const long long x = x0 + t;
            long long own = 0;
            if (x < tiles) {
                const int n = (int)(x / a.ktiles);
                const WindowLens len = {p.QLens ? min(max(p.QLens[n], 0), p.QL) : p.QL, p.VLens ? min(max(p.VLens[n], 0), p.VL) : p.VL};
                own = (long long)window_steps(window_queries(a, (int)(x - (long long)n * a.ktiles), len), 32) * group;
            }
            most = max(most, own);
            sum[t] = own;
            __syncthreads();
            for (int d = 1; d < NTHREADS; d <<= 1) {
                const long long add = t >= d ? sum[t - d] : 0;
                __syncthreads();
                sum[t] += add;
                __syncthreads();
            }
            if (x < tiles) a.before[x] = base + sum[t] - own;
            base += sum[NTHREADS - 1];
            __syncthreads();
        }
        sum[t] = most;
        __syncthreads();
        for (int d = NTHREADS / 2; d > 0; d >>= 1) {
            if (t < d) sum[t] = max(sum[t], sum[t + d]);
            __syncthreads();
        }
        if (t == 0) {
            a.before[tiles] = base;
            a.before[tiles + 1] = sum[0];
        }
        return;
    }
    const long long row = (long long)blockIdx.x * (NTHREADS / 32) + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const long long nh = row / p.QL;
    const int n = (int)(nh / p.head), hd = (int)(nh - (long long)n * p.head), i = (int)(row - nh * p.QL);
    const int d = 4 * (threadIdx.x & 31);
    float sum = 0.0f;
    const int ql = p.QLens ? min(p.QLens[n], p.QL) : p.QL;
    if (i < ql && d < p.dv4) {
        const size_t at = n * p.y.n + hd * p.y.h + (size_t)i * p.y.l + d;
        const v4f g = *(const v4f*)(a.dY + at), y = *(const v4f*)(p.Y + at);
        sum = (g.x * y.x + g.y * y.y) + (g.z * y.z + g.w * y.w);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
    if ((threadIdx.x & 31) == 0) {
        a.stats[row] = i < ql ? p.Lse[row] : 0.0f;
        a.stats[a.rows + row] = sum;
    }
}

constexpr int GT = 512;

// P of a score and its row's lse.  The difference is formed in units of e and near 0 where P counts; the scores are not
// accumulated from -lse on, nor is lse brought to units of log2 beforehand: either costs up to |lse| 2^-24 in every P of the row.
__device__ __forceinline__ float probability(float s, float lse) { return __builtin_amdgcn_exp2f((s - lse) * MIX_LOG2E); }

// P handed from one wavefront to the other: 16 bytes per lane and result group
__device__ __forceinline__ void give(float* at, const v16f& e) {
#pragma unroll
    for (int q = 0; q < 4; q++) *(v4f*)(at + q * 256) = (v4f){e[4 * q], e[4 * q + 1], e[4 * q + 2], e[4 * q + 3]};
}
__device__ __forceinline__ void take(const float* at, v16f& e) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const v4f P = *(const v4f*)(at + q * 256);
#pragma unroll
        for (int w = 0; w < 4; w++) e[4 * q + w] *= P[w];
    }
}

// ---------------------------------------------------------------- dQ
template <int DB, int DC, int KB>
__global__ __launch_bounds__(GT, DB > 2 ? 2 : 4) void window_grad_q(const WindowGrad a) {
    constexpr int DW = DB * 32, NG = DC * 4, AK = KB * 32, TILE = AK * DW;
    const WindowParams& p = a.w;
    __shared__ __attribute__((aligned(1024))) float Ks[3 * TILE];
    __shared__ __attribute__((aligned(1024))) float Vs[3 * TILE];
    __shared__ __attribute__((aligned(16))) float Ps[2][4][KB * 64 * 16];  // [step][32 queries][keys / 8][lane]
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const int block = wave & 3;
    const bool second = wave >= 4;
    const WindowJob job = window_job(p, blockIdx.x);
    const WindowLens len = window_lens(p, job.n);
    const int group = p.head / p.kv_head, off = len.vl - len.ql;
    const int row0 = job.qt * GQ, wrow = row0 + block * 32;
    const WindowRow row = window_row(p, job, wrow + r, group, len.ql);
    const size_t stat = ((size_t)job.n * p.head + row.hd) * p.QL + row.i;
    const WindowSpan all = window_span(row0, GQ, group, len.ql, off), span = window_span(wrow, 32, group, len.ql, off);
    const WindowRange range = window_range(p, all.first, all.last, all.first <= all.last, len.vl);
    const int nsink = (range.sink_end + AK - 1) / AK, steps = nsink + (max(range.hi - range.low, 0) + AK - 1) / AK;
    const bool live = row.live;
    const int pos = live ? row.i + off : -1;
    const int w0 = span.first, w1 = span.last;                          // the wavefront's positions

    v4f own[NG];                                                        // Q (times scale) or dY
    if (second) {
        mix_load_cols<NG>(own, a.dY + job.n * p.y.n + row.hd * p.y.h + (size_t)row.i * p.y.l, live, p.dv4, h);
    } else {
        mix_load_cols<NG>(own, p.Q + job.n * p.q.n + row.hd * p.q.h + (size_t)row.i * p.q.l, live, p.dk4, h);
#pragma unroll
        for (int g = 0; g < NG; g++) own[g] *= a.scale;
    }
    const float own_stat = live ? a.stats[(second ? a.rows : 0) + stat] : 0.0f;            // lse or D

    const float* Kb = p.K + job.n * p.k.n + job.kvh * p.k.h;
    const float* Vb = p.V + job.n * p.v.n + job.kvh * p.v.h;
    MixTile<DW, AK, true, GT> kt, vt;
    MixColumns<DW, true> cols;
    cols.init(r, h);
    kt.init(t, p.k.l, p.dk4);
    vt.init(t, p.v.l, p.dv4);
    const unsigned klds = mix_lds(Ks) + wave * 1024, vlds = mix_lds(Vs) + wave * 1024;
    const float* const X = second ? Vs : Ks;
    auto key_of = [&](int s) { return s < nsink ? s * AK : range.low + (s - nsink) * AK; };
    auto fetch = [&](int s, int into) {
        const int key0 = key_of(s), left = (s < nsink ? range.sink_end : range.hi) - key0;
        kt.fetch(Kb + (size_t)key0 * p.k.l, left, p.k.l, klds + into * (TILE * 4), wave);
        vt.fetch(Vb + (size_t)key0 * p.v.l, left, p.v.l, vlds + into * (TILE * 4), wave);
    };
    v16f o[DC];
#pragma unroll
    for (int b = 0; b < DC; b++) o[b] = (v16f)(0.0f);
    const int first = (int)((long long)steps * job.part / p.parts), last = (int)((long long)steps * (job.part + 1) / p.parts);
    if (first < last) fetch(first, 0);
    mix_wait();
    if (first + 1 < last) fetch(first + 1, 1);
    __syncthreads();
    int buf = 0;
    for (int s = first; s < last; s++) {
        const int key0 = key_of(s), limit = s < nsink ? range.sink_end : range.hi, end = min(key0 + AK, limit);
        const bool sees = w0 <= w1 && (s < nsink || (key0 <= w1 && (end - 1 > w0 - p.window || key0 < p.sinks)));
        float* exchange = &Ps[s & 1][block][4 * lane];
        v16f e[KB];
        if (sees) {
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                e[kb] = (v16f)(0.0f);
                mix_rows_product<DW, NG>(e[kb], X + buf * TILE + kb * 32 * DW, own, r, h);
            }
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int v = 0; v < 16; v++) e[kb][v] = second ? e[kb][v] - own_stat : probability(e[kb][v], own_stat);
            // keys behind a query (or behind the last key), and before its window: tested only where some query has them.
            // Both factors are cleared: dY.V^T may be anything where nothing is seen.
            if (key0 + AK - 1 > w0 || key0 + AK > limit || !span.full) {
                const int top = min(pos, limit - 1) - key0 - 4 * h;
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (32 * kb + mix_row(v, 0) > top) e[kb][v] = 0.0f;
            }
            if (s >= nsink && key0 <= w1 - p.window) {
                const int low = pos - p.window - key0 - 4 * h, sink = p.sinks - key0 - 4 * h;
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (32 * kb + mix_row(v, 0) <= low && 32 * kb + mix_row(v, 0) >= sink) e[kb][v] = 0.0f;
            }
            if (!second) {
#pragma unroll
                for (int kb = 0; kb < KB; kb++) give(exchange + kb * 1024, e[kb]);
            }
        }
        mix_wait();
        __syncthreads();
        const int b1 = buf == 2 ? 0 : buf + 1, b2 = b1 == 2 ? 0 : b1 + 1;
        if (s + 2 < last) fetch(s + 2, b2);
        __builtin_amdgcn_sched_barrier(0);
        if (sees && second) {
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                take(exchange + kb * 1024, e[kb]);
                mix_columns_product<DW, DC, true>(o, Ks + buf * TILE + kb * 32 * DW, e[kb], cols);
            }
        }
        buf = b1;
    }
    if (second && row.exists) {
        float* const out = p.parts == 1 ? a.dQ + job.n * p.q.n + row.hd * p.q.h + (size_t)row.i * p.q.l
                                        : p.part + (stat * p.parts + job.part) * p.dk4;
        mix_store_row<DC>(out, o, p.parts == 1 ? a.scale : 1.0f, p.dk4, h);
    }
}
// dQ from the parts that the keys were cut into, in order: 4 floats a thread
__device__ __forceinline__ void window_grad_join_q(const WindowGrad& a, long long x) {
    const WindowParams& p = a.w;
    const int per = p.dk4 / 4;
    const long long row = x / per;
    if (row >= a.rows) return;
    const int d = 4 * (int)(x - row * per), i = (int)(row % p.QL), hd = (int)(row / p.QL % p.head);
    const long long n = row / p.QL / p.head;
    const float* const part = p.part + row * p.parts * p.dk4 + d;
    v4f s = *(const v4f*)part;
#pragma unroll 4
    for (int k = 1; k < p.parts; k++) s += *(const v4f*)(part + (size_t)k * p.dk4);
    *(v4f*)(a.dQ + n * p.q.n + hd * p.q.h + (size_t)i * p.q.l + d) = s * a.scale;
}

// ---------------------------------------------------------------- dK, dV
// A key tile is seen by window + 128 queries of every head of the group, the last ones and those under no window by fewer or
// by more (and a tile of many sinks by all behind it): the tiles differ by whatever the sequence is long.  So the steps of all tiles are counted through
// (before) and dealt to the workgroups in equal runs.  Where a run begins or ends inside a tile the workgroup leaves its sums
// as a piece and window_grad_join adds the tile's pieces in order.
// Where there are no more tiles than workers and the largest exceeds a compute unit's share by no more than what the cuts cost
// -- about 5 steps -- every worker takes a tile: 512 tiles of 64 columns and 12 steps in 114 us instead of 127 (and the join
// in 7 instead of 12), 256 of 128 columns 263 us instead of 294 with everything around them.  But 256 tiles of 4 to 32 steps:
// 308 instead of 287.
constexpr int UNITS = 256, CUT_STEPS = 5;
struct GradDeal { long long total; long long workers; bool each; };
__device__ __forceinline__ GradDeal grad_deal(const WindowGrad& a) {
    const long long tiles = (long long)a.w.N * a.ktiles, all = tiles * a.w.kv_head;
    GradDeal x;
    x.total = a.before[tiles] * a.w.kv_head;
    x.each = all <= a.workers && a.before[tiles + 1] * (all > UNITS ? 2 : 1) <= x.total / UNITS + CUT_STEPS;
    x.workers = x.each ? all : min((long long)a.workers, max(x.total / 4, 1LL));     // at least 4 steps each
    return x;
}
// a tile in the count: its steps for one key / value head, where the heads' steps begin
struct GradTile { long long at; int steps; };
__device__ __forceinline__ GradTile grad_tile(const WindowGrad& a, long long tile) {
    GradTile x;
    x.at = a.before[tile] * a.w.kv_head;
    x.steps = (int)(a.before[tile + 1] - a.before[tile]);
    return x;
}
// the tile (over all sequences) that step `pos` of the count belongs to: the last one that begins at or before it
__device__ __forceinline__ long long grad_find(const WindowGrad& a, long long pos) {
    long long lo = 0, hi = (long long)a.w.N * a.ktiles;
    while (hi - lo > 1) {
        const long long mid = (lo + hi) >> 1;
        if (a.before[mid] * a.w.kv_head <= pos) lo = mid;
        else hi = mid;
    }
    return lo;
}
// where worker w's run begins; a boundary that is not farther from a tile's than what two pieces cost moves there
__device__ __forceinline__ long long grad_begin(const WindowGrad& a, const GradDeal& d, long long w) {
    if (w <= 0) return 0;
    if (w >= d.workers) return d.total;
    if (d.each) {
        const GradTile tile = grad_tile(a, w / a.w.kv_head);
        return tile.at + (w % a.w.kv_head) * tile.steps;
    }
    const long long pos = d.total / d.workers * w + (d.total % d.workers) * w / d.workers;
    const GradTile tile = grad_tile(a, grad_find(a, pos));
    if (tile.steps == 0) return pos;
    const int in = (int)((pos - tile.at) % tile.steps), snap = (int)min((long long)a.snap, d.total / d.workers / 2);
    return in <= snap ? pos - in : tile.steps - in <= snap ? pos + tile.steps - in : pos;
}
// the kernel's arguments, as if they had just been passed
__device__ __forceinline__ const WindowGrad& anew(const WindowGrad&) {
    auto at = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const WindowGrad*)(const char*)at;
}

template <int DB, int DC>
__global__ __launch_bounds__(GT, DB > 2 ? 2 : 4) void window_grad_kv(const WindowGrad arg) {
    constexpr int DW = DB * 32, NG = DC * 4, TILE = 32 * DW;
    __shared__ __attribute__((aligned(1024))) float Qs[3 * TILE];
    __shared__ __attribute__((aligned(1024))) float Gs[3 * TILE];
    __shared__ __attribute__((aligned(16))) float Ps[2][4][64 * 16];       // [step][32 keys][4 results][lane]
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const int block = wave & 3;
    const bool second = wave >= 4;

    const GradDeal deal = grad_deal(arg);
    auto uniform = [](long long x) { return (long long)(((unsigned long long)(unsigned)mix_uniform((int)(x >> 32)) << 32) | (unsigned)mix_uniform((int)x)); };
    if (blockIdx.x >= deal.workers) return;
    long long pos = uniform(grad_begin(arg, deal, blockIdx.x));
    const long long stop = uniform(grad_begin(arg, deal, blockIdx.x + 1));

    MixTile<DW, 32, true, GT> qt, gt;
    MixColumns<DW, true> cols;
    cols.init(r, h);
    qt.init(t, arg.w.q.l, arg.w.dk4);
    gt.init(t, arg.w.y.l, arg.w.dv4);
    const unsigned qlds = mix_lds(Qs) + wave * 1024, glds = mix_lds(Gs) + wave * 1024;
    const float* const X = second ? Gs : Qs;                            // the tile of the first product, of the second
    const float* const Z = second ? Qs : Gs;

    long long at = pos < stop ? uniform(grad_find(arg, pos)) : 0;         // the tile over all sequences
    while (pos < stop) {
        // The arguments are read anew for every piece: kept in scalar registers all through the kernel they do not fit there,
        // and under that pressure the compiler gives up the order of reads and matrix instructions in the loop below.
        const WindowGrad& a = anew(arg);
        const WindowParams& p = a.w;
        const int group = mix_uniform(p.head / p.kv_head);
        const float* const stats = a.stats + (second ? a.rows : 0);
        GradTile cur = grad_tile(a, at);
        while (pos >= cur.at + (long long)cur.steps * p.kv_head) cur = grad_tile(a, ++at);     // also over tiles without steps
        at = uniform(at);
        const int all = mix_uniform(cur.steps), kvh = mix_uniform((int)((pos - cur.at) / cur.steps));
        const int first = mix_uniform((int)(pos - cur.at - (long long)kvh * all));
        const int last = mix_uniform((int)min((long long)all, first + (stop - pos)));
        pos += last - first;
        const int n = mix_uniform((int)(at / a.ktiles)), tile = mix_uniform((int)(at - (long long)n * a.ktiles));
        const WindowLens len = window_lens(p, n);
        const WindowQueries qs = window_queries(a, tile, len);
        const int lo = qs.lo, hi = qs.hi, per_head = window_steps(qs, 32), off = len.vl - len.ql;
        const int u0 = tile * GK + block * 32, u1 = min(u0 + 32, len.vl) - 1;      // the wavefront's keys
        const int key = u0 + r;
        const bool live = key < len.vl;

        v4f own[NG];                                                    // K (times scale) or V
        if (second) {
            mix_load_cols<NG>(own, p.V + n * p.v.n + kvh * p.v.h + (size_t)min(key, p.VL - 1) * p.v.l, live, p.dv4, h);
        } else {
            mix_load_cols<NG>(own, p.K + n * p.k.n + kvh * p.k.h + (size_t)min(key, p.VL - 1) * p.k.l, live, p.dk4, h);
#pragma unroll
            for (int g = 0; g < NG; g++) own[g] *= a.scale;
        }
        // Queries go by in steps of 32 rows, head by head.  Everything that is fetched for a step moves along as an address (a
        // step on, or to the next head's first): so few scalar registers that the compiler keeps the loop's order.
        const int g0 = mix_uniform(first / per_head);
        int i0 = lo + (first - g0 * per_head) * 32;                     // the step's queries
        struct Walk {
            int i0;
            const float* at;
            __device__ __forceinline__ void next(int lo, int hi, int step, long long jump) {
                i0 += 32;
                if (i0 >= hi) { i0 = lo; at += jump; }
                else at += step;
            }
        };
        const int hd0 = kvh * group + g0;
        Walk wq = {i0, p.Q + n * p.q.n + hd0 * p.q.h + (size_t)i0 * p.q.l};
        Walk wg = {i0, a.dY + n * p.y.n + hd0 * p.y.h + (size_t)i0 * p.y.l};
        Walk ws = {i0, stats + ((size_t)n * p.head + hd0) * p.QL + i0};
        const long long q_jump = p.q.h - (long long)(per_head - 1) * 32 * p.q.l, g_jump = p.y.h - (long long)(per_head - 1) * 32 * p.y.l;
        const int s_jump = p.QL - (per_head - 1) * 32;
        auto fetch = [&](int into) {
            qt.fetch(wq.at, hi - wq.i0, p.q.l, qlds + into * (TILE * 4), wave);
            gt.fetch(wg.at, hi - wq.i0, p.y.l, glds + into * (TILE * 4), wave);
            wg.next(lo, hi, 32 * p.y.l, g_jump);
            wq.next(lo, hi, 32 * p.q.l, q_jump);
        };
        // lse or D of a step's queries: rows 8q + 4h .. +3 (zeros beyond the last of the sequence)
        v16f stat;
        auto begin = [&]() {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)ws.at, 0, min(hi - ws.i0, 32) * 4, RSRC_FLAGS);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const v4f x = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rs, (8 * q + 4 * h) * 4, 0, 0));
#pragma unroll
                for (int w = 0; w < 4; w++) stat[4 * q + w] = x[w];
            }
            ws.next(lo, hi, 32, s_jump);
        };
        v16f acc[DC];
#pragma unroll
        for (int b = 0; b < DC; b++) acc[b] = (v16f)(0.0f);

        fetch(0);
        begin();
        mix_wait();
        if (first + 1 < last) fetch(1);
        __syncthreads();
        int buf = 0;
        for (int s = first; s < last; s++) {
            const int p0 = i0 + off, p1 = min(i0 + 32, hi) - 1 + off;  // the step's positions
            const bool sees = u0 <= u1 && p1 >= u0 && (p0 < u1 + p.window || u0 < p.sinks);
            float* exchange = &Ps[s & 1][block][4 * lane];
            v16f e = (v16f)(0.0f);
            if (sees) {
                mix_rows_product<DW, NG>(e, X + buf * TILE, own, r, h);
#pragma unroll
                for (int v = 0; v < 16; v++) e[v] = second ? e[v] - stat[v] : probability(e[v], stat[v]);
                // queries before a key, those whose window has passed it, and rows behind the last: tested only where there are
                // any.  Both factors are cleared: dY.V^T may be anything where nothing is seen.
                if (p0 < u1 || i0 + 32 > hi || u0 + 32 > len.vl) {
                    const int low = (live ? key : 0x3fffffff) - p0 - 4 * h, top = hi - 1 - i0 - 4 * h;
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (mix_row(v, 0) < low || mix_row(v, 0) > top) e[v] = 0.0f;
                }
                if (p1 >= u0 + p.window) {
                    const int top = key < p.sinks ? 0x3fffffff : key + p.window - 1 - p0 - 4 * h;
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (mix_row(v, 0) > top) e[v] = 0.0f;
                }
                if (!second) give(exchange, e);
            }
            mix_wait();
            __syncthreads();
            const int b1 = buf == 2 ? 0 : buf + 1, b2 = b1 == 2 ? 0 : b1 + 1;
            if (s + 1 < last) begin();                                  // needed behind the next step's first product
            if (s + 2 < last) fetch(b2);
            __builtin_amdgcn_sched_barrier(0);
            if (sees) {
                if (second) take(exchange, e);
                mix_columns_product<DW, DC, true>(acc, Z + buf * TILE, e, cols);
            }
            buf = b1;
            i0 += 32;
            if (i0 >= hi) i0 = lo;
        }
        const WindowGrad& b = anew(arg);
        if (t == 0) {
            int2* cut = b.cut + at * b.w.kv_head + kvh;
            if (first == 0) cut->x = blockIdx.x;
            if (last == all) cut->y = blockIdx.x;
        }
        float* out;
        if (first == 0 && last == all) {
            out = second ? b.dK + n * b.w.k.n + kvh * b.w.k.h + (size_t)key * b.w.k.l : b.dV + n * b.w.v.n + kvh * b.w.v.h + (size_t)key * b.w.v.l;
        } else {        // a piece that does not begin the tile is this run's first, one that does its last
            out = b.pieces + ((2 * (size_t)blockIdx.x + (first == 0)) * GK + block * 32 + r) * (b.w.dk4 + b.w.dv4) + (second ? 0 : b.w.dk4);
        }
        if (key < b.w.VL) mix_store_row<DC>(out, acc, second ? b.scale : 1.0f, second ? b.w.dk4 : b.w.dv4, h);
        __syncthreads();                                                // the next piece's first tile lands in buffer 0
    }
}

// ---------------------------------------------------------------- dK, dV of the sinks
// What the queries beyond a sink's window leave there: all of them, for a few keys, so the reading of Q and dY bounds it and
// not the products.  16 keys a workgroup, SINK_QUERIES queries of every head of the group, 16 at a time per wavefront, with
// v_mfma_f32_16x16x4_f32 and the register layouts of window_rows (queries and keys changed about): a lane reads a query's row
// once in pieces for the scores and once as the columns of the sums.  (In tiles of 128 keys like the rest, three of four
// wavefronts have nothing to do: at 4 sinks and 8192 queries a tenth of window_grad_kv's steps.)  32 heads of 128 and 8192
// queries in 76 us, 3.5 TB/s.
constexpr int SINK_QUERIES = 128;
template <int DE>
__global__ __launch_bounds__(NTHREADS, 2) void window_grad_sinks(const WindowGrad a) {
    constexpr int NS = DE * 4;
    const WindowParams& p = a.w;
    __shared__ __attribute__((aligned(16))) float So[4][16][DE * 64 + 4];
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), c = lane & 15, k4 = lane >> 4;
    const int nkv = p.N * p.kv_head, group = p.head / p.kv_head;
    const int x = mix_uniform(blockIdx.x / nkv), kv = blockIdx.x - x * nkv;
    const int part = mix_uniform(x / a.sink_blocks), block = x - part * a.sink_blocks;
    const int n = mix_uniform(kv / p.kv_head), kvh = kv - n * p.kv_head;
    const WindowLens len = window_lens(p, n);
    const int key = block * 16 + c, keys = min(p.sinks, len.vl);
    const bool live = key < keys;
    // behind the queries that the tile of 128 keys walks over (none of them where they all lie beyond its window: hi < 0)
    const int lo = max(window_queries(a, block * 16 / GK, len).hi, 0) + part * SINK_QUERIES;
    const int hi = block * 16 < keys ? min(lo + SINK_QUERIES, len.ql) : 0;

    v4f kf[NS], vf[NS];
    const float* krow = p.K + n * p.k.n + kvh * p.k.h + (size_t)min(key, p.VL - 1) * p.k.l;
    const float* vrow = p.V + n * p.v.n + kvh * p.v.h + (size_t)min(key, p.VL - 1) * p.v.l;
    int qa[NS], ga[NS], qc[4 * DE], gc[4 * DE];               // byte offsets inside 16 rows
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const int d = 16 * s + 4 * k4;
        kf[s] = (live && d < p.dk4) ? *(const v4f*)(krow + d) * a.scale : (v4f)(0.0f);
        vf[s] = (live && d < p.dv4) ? *(const v4f*)(vrow + d) : (v4f)(0.0f);
        qa[s] = d < p.dk4 ? (c * p.q.l + d) * 4 : OOB_OFFSET;
        ga[s] = d < p.dv4 ? (c * p.y.l + d) * 4 : OOB_OFFSET;
    }
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
        for (int e = 0; e < DE; e++) {
            const int d = 64 * e + 4 * c;
            qc[v * DE + e] = d < p.dk4 ? ((4 * k4 + v) * p.q.l + d) * 4 : OOB_OFFSET;
            gc[v * DE + e] = d < p.dv4 ? ((4 * k4 + v) * p.y.l + d) * 4 : OOB_OFFSET;
        }
    v4f dk[DE][4], dv[DE][4];
#pragma unroll
    for (int e = 0; e < DE; e++)
#pragma unroll
        for (int u = 0; u < 4; u++) dk[e][u] = dv[e][u] = (v4f)(0.0f);
    for (int g = 0; g < group; g++) {
        const int hd = kvh * group + g;
        const float* qb = p.Q + n * p.q.n + hd * p.q.h;
        const float* gb = a.dY + n * p.y.n + hd * p.y.h;
        const float* sb = a.stats + ((size_t)n * p.head + hd) * p.QL;
        for (int i0 = lo + 16 * wave; i0 < hi; i0 += 64) {
            const int left = min(hi - i0, 16);
            const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)(qb + (size_t)i0 * p.q.l), 0, left * p.q.l * 4, RSRC_FLAGS);
            const __amdgpu_buffer_rsrc_t rg = __builtin_amdgcn_make_buffer_rsrc((void*)(gb + (size_t)i0 * p.y.l), 0, left * p.y.l * 4, RSRC_FLAGS);
            const __amdgpu_buffer_rsrc_t rl = __builtin_amdgcn_make_buffer_rsrc((void*)(sb + i0), 0, left * 4, RSRC_FLAGS);
            const __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)(sb + a.rows + i0), 0, left * 4, RSRC_FLAGS);
            const v4f lse = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rl, 16 * k4, 0, 0));
            const v4f D = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rd, 16 * k4, 0, 0));
            v4f s = (v4f)(0.0f), d = (v4f)(0.0f);
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const v4f q = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rq, qa[i], 0, 0));
                const v4f y = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rg, ga[i], 0, 0));
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    s = __builtin_amdgcn_mfma_f32_16x16x4f32(q[u], kf[i][u], s, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x4f32(y[u], vf[i][u], d, 0, 0, 0);
                }
            }
            // register v: query i0 + 4 * k4 + v
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const bool on = live && 4 * k4 + v < left;
                s[v] = on ? probability(s[v], lse[v]) : 0.0f;
                d[v] = on ? s[v] * (d[v] - D[v]) : 0.0f;
            }
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int e = 0; e < DE; e++) {
                    const v4f y = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rg, gc[v * DE + e], 0, 0));
                    const v4f q = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rq, qc[v * DE + e], 0, 0));
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        dv[e][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[u], s[v], dv[e][u], 0, 0, 0);
                        dk[e][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[u], d[v], dk[e][u], 0, 0, 0);
                    }
                }
        }
    }
    // the wavefronts' sums, added through LDS; register w of block (e, u) is float 64e + 16*k4 + 4w + u of key c
    float* out = a.sinks + (((size_t)kv * a.sink_blocks + block) * a.sink_parts + part) * 16 * (p.dk4 + p.dv4);
    auto join = [&](const v4f (&o)[DE][4], int at, int d4, float f) {
#pragma unroll
        for (int e = 0; e < DE; e++)
#pragma unroll
            for (int w = 0; w < 4; w++)
                *(v4f*)&So[wave][c][64 * e + 16 * k4 + 4 * w] = (v4f){o[e][0][w], o[e][1][w], o[e][2][w], o[e][3][w]};
        __syncthreads();
        for (int i = t; i < 4 * d4; i += NTHREADS) {
            const int row = i / (d4 / 4), d = 4 * (i - row * (d4 / 4));
            const v4f sum = (*(const v4f*)&So[0][row][d] + *(const v4f*)&So[1][row][d]) + (*(const v4f*)&So[2][row][d] + *(const v4f*)&So[3][row][d]);
            *(v4f*)(out + (size_t)row * (p.dk4 + p.dv4) + at + d) = sum * f;
        }
        __syncthreads();
    };
    join(dk, 0, p.dk4, a.scale);
    join(dv, p.dk4, p.dv4, 1.0f);
}

// ---------------------------------------------------------------- everything that a key's gradient is made of
// Four workgroups per tile and key / value head: the tile's pieces in order, or what was written whole, or zeros where no
// query sees it; then the sinks' parts in order.  The workgroups behind them join dQ where the keys were cut.
__global__ __launch_bounds__(NTHREADS) void window_grad_join(const WindowGrad a) {
    const WindowParams& p = a.w;
    const long long at = blockIdx.x / p.kv_head;
    if (at >= (long long)p.N * a.ktiles) {
        window_grad_join_q(a, ((blockIdx.x - (long long)p.N * a.ktiles * p.kv_head) * 4 + blockIdx.y) * NTHREADS + threadIdx.x);
        return;
    }
    const int kvh = (int)(blockIdx.x - at * p.kv_head), n = (int)(at / a.ktiles), k0 = (int)(at - (long long)n * a.ktiles) * GK;
    const bool some = a.before[at + 1] != a.before[at];
    const int2 cut = some ? a.cut[at * p.kv_head + kvh] : make_int2(0, 0);
    const bool whole = some && cut.x == cut.y;
    if (whole && k0 >= a.sink_blocks * 16) return;
    const int width = p.dk4 + p.dv4, per = width / 4;
    for (int x = threadIdx.x; x < GK / 4 * per; x += NTHREADS) {
        const int in = x / per, row = blockIdx.y * (GK / 4) + in, d = 4 * (x - in * per), key = k0 + row;
        if (key >= p.VL || (whole && key >= a.sink_blocks * 16)) break;
        float* out = d < p.dk4 ? a.dK + n * p.k.n + kvh * p.k.h + (size_t)key * p.k.l + d
                               : a.dV + n * p.v.n + kvh * p.v.h + (size_t)key * p.v.l + d - p.dk4;
        v4f s = (v4f)(0.0f);
        if (whole) {
            s = *(const v4f*)out;
        } else if (some) {
            s = *(const v4f*)(a.pieces + ((2 * (size_t)cut.x + 1) * GK + row) * width + d);
#pragma unroll 4
            for (int w = cut.x + 1; w <= cut.y; w++) s += *(const v4f*)(a.pieces + (2 * (size_t)w * GK + row) * width + d);
        }
        if (key < a.sink_blocks * 16) {
            const int block = key / 16;
            const float* parts = a.sinks + (((size_t)(n * p.kv_head + kvh) * a.sink_blocks + block) * a.sink_parts * 16 + (key - block * 16)) * width + d;
#pragma unroll 8
            for (int i = 0; i < a.sink_parts; i++) s += *(const v4f*)(parts + (size_t)i * 16 * width);
        }
        *(v4f*)out = s;
    }
}

// ---------------------------------------------------------------- host side
// Cuts of the keys of window_grad_q: where the tiles are few, several workgroups walk over a tile's keys, at least 2 steps each,
// and window_grad_join adds their sums in order (7 x 1023 queries of one head of 112: 198 -> 50 us; one head of 4096 of 64:
// 430 -> 47).  Few is half of what the compute units hold under a window, all of it where the tiles see everything before
// them and differ by the sequence: cut there, 256 tiles of 64 take 303 us with everything around them instead of 332, but 184
// -> 187 under a window of 256; cut for twice as many, 192 tiles of 128 take 404 us instead of 393.
int window_grad_parts(int N, int head, int kv_head, int QL, int VL, int workers, int window, int sinks) {
    const long long group = head / kv_head, base = (long long)N * kv_head * ((QL * group + GQ - 1) / GQ);
    const long long reach = window == 0 ? VL : (long long)window + sinks + (GQ + group - 1) / group;
    const long long steps = ((reach < VL ? reach : VL) + 31) / 32;
    long long parts = base >= (reach < VL ? workers / 2 : workers) ? 1 : (workers + base - 1) / base;
    if (parts > steps / 2) parts = steps / 2;
    return (int)(parts < 1 ? 1 : parts);
}
// The caller's buffer, in floats: the statistics, the running sum (64-bit), the pieces and whose they are, the sinks' parts,
// the parts of dQ.
// Up to here window_grad_sinks takes the queries beyond the window.  Training 4 x 1024, 16 heads of 64 under a window of 256: with 4
// sinks 294 us (in the tiles 334), with 64 325 (342), with 100 367 (363); 8192, 32 heads of 128 on 8 under 1024: with 4 sinks 5188
// (5350), with 64 5441 (5416), with 100 5754 (5546).
constexpr int SINKS_APART = 64;
// also the workgroups of every launch: rows' statistics, dQ, sinks, joins (window_grad_kv: the workers)
struct WindowGradBuffer {
    int ktiles, workers, qtiles, sink_blocks, sink_parts, parts;
    long long stats, before, pieces, cut, sinks, all;
    long long run_delta, run_q, run_sinks, run_join;
    bool fits;
};
WindowGradBuffer window_grad_buffer(int N, int head, int kv_head, int QL, int VL, int dk4, int dv4, int window, int sinks) {
    WindowGradBuffer b;
    b.ktiles = (VL + GK - 1) / GK;
    // as many workers as the compute units hold, or as there are tiles or runs of 4 steps
    const long long hold = (dk4 > dv4 ? dk4 : dv4) > 64 ? UNITS : 2 * UNITS, tiles = (long long)N * b.ktiles * kv_head;
    const long long runs = tiles * (head / kv_head) * ((QL + 31LL) / 32) / 4, most = tiles > runs ? tiles : runs;
    b.workers = (int)(most < hold ? most : hold);
    const bool apart = window != 0 && window < VL && sinks > 0 && sinks <= SINKS_APART;
    b.sink_blocks = apart ? ((sinks < VL ? sinks : VL) + 15) / 16 : 0;
    b.sink_parts = apart ? (QL + SINK_QUERIES - 1) / SINK_QUERIES : 0;
    b.stats = (2LL * N * head * QL + 3) / 4 * 4;
    b.before = (((long long)N * b.ktiles + 2) * 2 + 3) / 4 * 4;
    b.pieces = 2LL * b.workers * GK * (dk4 + dv4);
    b.cut = ((long long)N * b.ktiles * kv_head * 2 + 3) / 4 * 4;
    b.sinks = (long long)N * kv_head * b.sink_blocks * b.sink_parts * 16 * (dk4 + dv4);
    b.parts = window_grad_parts(N, head, kv_head, QL, VL, (int)hold, window, sinks);
    const long long rows = (long long)N * head * QL;
    b.all = b.stats + b.before + b.pieces + b.cut + b.sinks + (b.parts > 1 ? rows * b.parts * dk4 : 0);
    b.qtiles = (int)(((long long)QL * (head / kv_head) + GQ - 1) / GQ);
    b.run_delta = (rows + NTHREADS / 32 - 1) / (NTHREADS / 32) + 1;
    b.run_q = (long long)N * kv_head * b.qtiles * b.parts;
    b.run_sinks = (long long)N * kv_head * b.sink_blocks * b.sink_parts;
    b.run_join = tiles + (b.parts == 1 ? 0 : (rows * (dk4 / 4) + 4 * NTHREADS - 1) / (4 * NTHREADS));
    b.fits = mix_launch_fits(b.run_delta, NTHREADS) && mix_launch_fits(b.run_q, GT) && mix_launch_fits(b.run_sinks, NTHREADS) &&
             mix_launch_fits(b.run_join, NTHREADS);
    return b;
}

}  // namespace
}  // namespace dragon

using namespace dragon;

extern "C" {

int64_t dragon_Cuda_attention_window_backward_bufsize(int32_t N, int32_t head, int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4,
                                                      int32_t dV4, int32_t window, int32_t sinks) {
    if (!window_arguments_ok(N, head, kv_head, QL, VL, dK4, dV4, window, sinks)) return -1;
    const WindowGradBuffer b = window_grad_buffer(N, head, kv_head, QL, VL, dK4, dV4, window, sinks);
    return b.fits ? b.all * 4 : -1;
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
    const WindowGradBuffer b = window_grad_buffer(N, head, kv_head, QL, VL, dK4, dV4, window, sinks);
    const long long need = b.all * 4;
    if (!b.fits) return hipErrorInvalidValue;
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
    p.qtiles = b.qtiles; p.parts = b.parts;
    a.dY = (const float*)(intptr_t)dDeltaY;
    a.dQ = (float*)(intptr_t)dDeltaQ; a.dK = (float*)(intptr_t)dDeltaK; a.dV = (float*)(intptr_t)dDeltaV;
    a.stats = (float*)(intptr_t)dBuf;
    a.rows = (long long)N * head * QL;
    a.scale = scale;
    a.ktiles = b.ktiles; a.workers = b.workers;
    a.snap = 2;     // (0: level on seven shapes but 294 us for 302 on 3 ragged 1500; 5: 2 to 6 % slower wherever tiles are cut)
    a.before = (long long*)(a.stats + b.stats);
    a.pieces = a.stats + b.stats + b.before;
    a.cut = (int2*)(a.pieces + b.pieces);
    a.sinks = a.pieces + b.pieces + b.cut;
    p.part = a.sinks + b.sinks;
    a.sink_blocks = b.sink_blocks; a.sink_parts = b.sink_parts;
    split_ledger_touch(a.dQ, (size_t)N * head * QL * dK4 * 4);
    split_ledger_touch(a.dK, (size_t)N * kv_head * VL * dK4 * 4);
    split_ledger_touch(a.dV, (size_t)N * kv_head * VL * dV4 * 4);
    split_ledger_touch(a.stats, (size_t)need);

    hipStream_t s = (hipStream_t)(intptr_t)streams[0];
    const dim3 block(NTHREADS);
    hipLaunchKernelGGL(window_delta, dim3((unsigned)b.run_delta), block, 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 gq((unsigned)b.run_q), gk((unsigned)b.workers);
    const int dmax = dK4 > dV4 ? dK4 : dV4;
#define GRAD_CASE(DB_, DC_, B_)                                                        \
    do {                                                                              \
        hipLaunchKernelGGL((window_grad_kv<DB_, DC_>), gk, dim3(GT), 0, s, a);        \
        e = hipGetLastError();                                                        \
        if (e != hipSuccess) return e;                                                \
        hipLaunchKernelGGL((window_grad_q<DB_, DC_, B_>), gq, dim3(GT), 0, s, a);         \
        e = hipGetLastError();                                                        \
        if (e != hipSuccess) return e;                                                \
    } while (0)
    switch ((dmax + 31) / 32) {
        case 1: GRAD_CASE(1, 1, 1); break;
        case 2: GRAD_CASE(2, 2, 1); break;
        case 3: GRAD_CASE(4, 3, 1); break;
        default: GRAD_CASE(4, 4, 1); break;
    }
#undef GRAD_CASE
    if (b.sink_blocks > 0) {
        const dim3 gs((unsigned)b.run_sinks);
        if (dmax <= 64) hipLaunchKernelGGL(window_grad_sinks<1>, gs, block, 0, s, a);
        else hipLaunchKernelGGL(window_grad_sinks<2>, gs, block, 0, s, a);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(window_grad_join, dim3((unsigned)b.run_join, 4), block, 0, s, a);
    e = hipGetLastError();
    return e;
}

}  // extern "C"
