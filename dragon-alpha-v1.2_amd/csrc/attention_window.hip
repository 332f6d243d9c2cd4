// Attention in which a query sees the keys up to its own position, of those only the last `window` (0: all) and the first
// `sinks`, with key / value heads that several query heads share, sequences of their own lengths in a padded batch, and
// fewer queries than keys (the queries are the LAST ones of the sequence: a prompt's next piece, a single token on a cache):
//     position(i) = i + vl - ql;   i sees j  <=>  i < ql, j < vl, j <= position(i), (j > position(i) - window or j < sinks)
//     Y[i] = sum_j softmax_j(scale * <Q[i], K[j]>) * V[j] over the keys seen;   lse[i] = log sum_j exp(scale * <Q[i], K[j]>)
// A row that sees nothing (also the rows behind a sequence's queries) is zeros with lse = -infinity.
//
// Two kernels, chosen by the number of queries:
//   window_tiles: 128 (query, head) rows of one key / value head per workgroup, the keys they see in steps, S^T = K.Q^T and Y^T = V^T.P^T with
//     v_mfma_f32_32x32x2_f32 and a running maximum and sum per query (token_mixer.h has the register layouts).  The steps
//     are the sinks below the window's reach, then the keys from the first one that some query of the tile sees: no other
//     key is read.  Bound by the FP32 matrix pipe: 16384 queries of 8 heads of 128 under a window of 2048 in 1.01 ms, 128
//     TFLOP/s of what they see, the pipes busy for 83 % of the time (the rest: the softmax's vector instructions, the barrier).
//   window_rows: up to 16 (query, head) rows that share a key / value head per wavefront; keys and values go from memory
//     straight into v_mfma_f32_16x16x4_f32 operands, 16 keys at a time.  Bound by reading K and V: 64 sequences of 8 heads of
//     128 under a window of 4096 in 281 us, 5.8 TB/s.
// Where either leaves compute units idle the keys are cut: every part leaves its maximum, sum and un-normalised output in the
// caller's buffer and window_join adds them in order (a second launch, so the result does not depend on who is last).
#include "token_mixer.h"
#include "attention_window.h"
#include "runtime_internal.h"
#include "stream_policy.h"
#include "../../include/dragon_hip_gemm.h"
#include "../../include/dragon_hip_testing.h"

namespace dragon {
namespace {

constexpr int AQ = 128;          // rows per workgroup of the tiled kernel: 32 per wavefront
constexpr int LAG = 8;           // the reference maximum may lag the true one by 2^LAG
constexpr float NEG = -__builtin_inff();
constexpr float LOWEST = -3.402823466e38f;   // not above any score but -infinity

// ---------------------------------------------------------------- the keys cut into parts
// A launch has N * kv_head * qtiles * parts workgroups, from the capacities: `parts` for each tile.  Where the sequences have
// lengths window_tiles deals them by the steps that a tile has, so that the longest part is as short as can be: pieces of 500 and
// 250 on 9000 and 4500 keys of 16 heads of 96 in 305 us instead of 418, prompts of 1000 to 250 of 8 heads of 64 in 47 instead of
// 65.  Every wavefront works the deal out for itself, a pair (tile, sequence) a lane; the first workgroup of a pair writes it
// down for window_join.  (window_rows reads so little that the deal costs it more: 16.2 -> 17.8 us at 8 sequences of up to 4096.
// Nothing is dealt where the sizes alone fill the chip: there a long sequence among short ones keeps its own workgroups busy.)
constexpr int PAIRS = 512;      // at most, where there are parts (window_plan)
struct WindowCutting {
    int per, ak, least, want;   // rows of a tile, keys of a step, steps worth a part, workgroups on the chip
    bool deal;                  // parts by length
};
constexpr WindowCutting ROWS_CUTTING = {16, 16, 8, 256, false};
__host__ __device__ constexpr WindowCutting tile_cutting(int ak, bool deal) { return {AQ, ak, 4, 512, deal}; }

// the steps of pair x = (qtiles - 1 - tile) * N + sequence: tiles at the sequences' ends first
__device__ __forceinline__ int window_pair_steps(const WindowParams& p, const WindowCutting& c, int x) {
    const int q = x / p.N, n = x - q * p.N, row0 = (p.qtiles - 1 - q) * c.per, group = p.head / p.kv_head;
    const int ql = p.QLens ? min(max(p.QLens[n], 0), p.QL) : p.QL, vl = p.VLens ? min(max(p.VLens[n], 0), p.VL) : p.VL;
    const int end = min(row0 + c.per, ql * group), off = vl - ql;
    const WindowRange range = window_range(p, row0 / group + off, (end - 1) / group + off, end > row0, vl);
    return (range.sink_end + c.ak - 1) / c.ak + (max(range.hi - range.low, 0) + c.ak - 1) / c.ak;
}
// Between which numbers of steps the longest part is looked for, so that the pairs' parts fit the slots: with hi they do.  (A pair
// has at most one part more than its steps / longest, so all / (slots - pairs) is enough, and all / slots is needed; beside
// few spare slots the former leaves 32 bits where the keys are more than 10^8, so it ends at more steps than a tile can have.)
struct WindowDealBounds { int lo, hi; };
__host__ __device__ inline WindowDealBounds window_deal_bounds(double all, int slots, int pairs, int least) {
    constexpr int MOST = 0x3fffffff;
    const double enough = slots > pairs ? all / (slots - pairs) + 1.0 : (double)MOST;
    WindowDealBounds x;
    x.lo = max(least, (int)(all / slots));
    x.hi = max(enough < MOST ? (int)enough : MOST, x.lo);
    return x;
}
// sum over this lane and those below it
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);      // the lane 1 below, in rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // the last lane of row 0 to row 1, of 2 to 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // of row 1 to rows 2 and 3
    return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// what a part's row leaves: its output, its (maximum, sum); behind them {first slot, parts} of every pair
__device__ __forceinline__ float* window_part_o(const WindowParams& p, const WindowCutting& c, int slot, int row) {
    return p.part + ((size_t)slot * c.per + row) * p.dv4;
}
__device__ __forceinline__ float2& window_part_ml(const WindowParams& p, const WindowCutting& c, int slot, int row) {
    return ((float2*)(p.part + (size_t)p.N * p.kv_head * p.qtiles * p.parts * c.per * p.dv4))[(size_t)slot * c.per + row];
}
__device__ __forceinline__ int2& window_part_deal(const WindowParams& p, const WindowCutting& c, int pair) {
    return ((int2*)(p.part + (size_t)p.N * p.kv_head * p.qtiles * p.parts * c.per * (p.dv4 + 2)))[pair];
}

// a workgroup's tile and its part of that tile's keys; slot: where its results go.  none: a workgroup too many
struct WindowPart { WindowJob job; int parts, slot; bool none; };
__device__ __forceinline__ WindowPart window_part(const WindowParams& p, const WindowCutting c, int id) {
    WindowPart x;
    x.parts = p.parts;
    x.slot = 0;
    x.none = false;
    const int pairs = p.N * p.qtiles, lane = threadIdx.x & 63;
    if (!c.deal) {
        x.job = window_job(p, id);
        x.slot = (x.job.kvh * pairs + (p.qtiles - 1 - x.job.qt) * p.N + x.job.n) * p.parts + x.job.part;
        return x;
    }
    const int slots = min(pairs * p.parts, c.want / p.kv_head), at = mix_uniform(id / p.kv_head);   // >= pairs (window_plan)
    int steps[PAIRS / 64];
#pragma unroll
    for (int k = 0; k < PAIRS / 64; k++) {
        steps[k] = 0;
        if (64 * k < pairs && 64 * k + lane < pairs) steps[k] = window_pair_steps(p, c, 64 * k + lane);
    }
    // the least `longest` for which the parts fit the slots (the steps' sum may be beyond 32 bits)
    double all = 0.0;
#pragma unroll
    for (int k = 0; k < PAIRS / 64; k++)
        if (64 * k < pairs) all += (double)wave_sum(steps[k] >> 12) * 4096.0 + (double)wave_sum(steps[k] & 4095);
    auto parts_of = [](int steps, int longest) { return max((int)((unsigned)(steps + longest - 1) / (unsigned)longest), 1); };
    const WindowDealBounds bounds = window_deal_bounds(all, slots, pairs, c.least);
    int lo = bounds.lo, hi = bounds.hi;
    while (lo < hi) {
        const int longest = (lo + hi) >> 1;
        int sum = 0;
#pragma unroll
        for (int k = 0; k < PAIRS / 64; k++)
            if (64 * k < pairs) sum += 64 * k + lane < pairs ? parts_of(steps[k], longest) : 0;
        if (wave_sum(sum) <= slots) hi = longest;
        else lo = longest + 1;
    }
    x.none = true;
    int base = 0;
#pragma unroll
    for (int k = 0; k < PAIRS / 64; k++) {
        if (64 * k < pairs && x.none) {
            const int own = 64 * k + lane < pairs ? parts_of(steps[k], hi) : 0, end = base + wave_scan(own);
            const unsigned long long behind = __ballot(end > at);
            if (behind != 0) {
                const int l = __builtin_ctzll(behind), pair = 64 * k + l, q = mix_uniform(pair / p.N);
                x.parts = __builtin_amdgcn_readlane(own, l);
                const int first = __builtin_amdgcn_readlane(end, l) - x.parts;
                x.job.part = at - first;
                x.job.qt = p.qtiles - 1 - q;
                x.job.n = pair - q * p.N;
                x.job.kvh = id - at * p.kv_head;
                x.slot = x.job.kvh * pairs * p.parts + at;
                x.none = false;
                if (threadIdx.x == 0 && x.job.kvh == 0 && x.job.part == 0) window_part_deal(p, c, pair) = make_int2(first, x.parts);
            }
            base = __builtin_amdgcn_readlane(end, 63);
        }
    }
    return x;
}

// ---------------------------------------------------------------- many queries
template <int DB, int DC, int KB, bool DEAL>
__global__ __launch_bounds__(NTHREADS, 2) void window_tiles(const WindowParams p) {
    constexpr int AK = KB * 32, DW = DB * 32, NG = DC * 4;
    constexpr WindowCutting cutting = tile_cutting(AK, DEAL);
    __shared__ __attribute__((aligned(1024))) float Ks[2][AK * DW];
    __shared__ __attribute__((aligned(1024))) float Vs[2][AK * DW];

    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const WindowPart part = window_part(p, cutting, blockIdx.x);
    if (part.none) return;
    const WindowJob job = part.job;
    const WindowLens len = window_lens(p, job.n);
    const int group = p.head / p.kv_head, off = len.vl - len.ql;
    const int row0 = job.qt * AQ, wrow = row0 + 32 * wave;
    const WindowRow row = window_row(p, job, wrow + r, group, len.ql);
    const size_t stat = ((size_t)job.n * p.head + row.hd) * p.QL + row.i;

    // the keys that the tile's rows see: [0, sink_end) and [low, hi)
    const WindowSpan all = window_span(row0, AQ, group, len.ql, off), span = window_span(wrow, 32, group, len.ql, off);
    const WindowRange range = window_range(p, all.first, all.last, all.first <= all.last, len.vl);
    const int nsink = (range.sink_end + AK - 1) / AK, nwin = (max(range.hi - range.low, 0) + AK - 1) / AK;
    const int first = mix_uniform((int)((long long)(nsink + nwin) * job.part / part.parts));
    const int last = mix_uniform((int)((long long)(nsink + nwin) * (job.part + 1) / part.parts));
    const int pos = row.live ? row.i + off : -1;
    const int w0 = span.first, w1 = span.last;              // the wavefront's positions

    v4f qf[NG];
    mix_load_cols<NG>(qf, p.Q + job.n * p.q.n + row.hd * p.q.h + (size_t)row.i * p.q.l, row.live, p.dk4, h);
#pragma unroll
    for (int g = 0; g < NG; g++) qf[g] *= p.c;              // scores in units of log2

    const float* Kb = p.K + job.n * p.k.n + job.kvh * p.k.h;
    const float* Vb = p.V + job.n * p.v.n + job.kvh * p.v.h;
    MixTile<DW, AK, true> kt;
    MixTile<DW, AK, false> vt;
    MixColumns<DW, false> vcols;
    vcols.init(r, h);
    kt.init(t, p.k.l, p.dk4);
    vt.init(t, p.v.l, p.dv4);
    auto key_of = [&](int s) { return s < nsink ? s * AK : range.low + (s - nsink) * AK; };
    const unsigned klds = mix_lds(Ks[0]) + wave * 1024, vlds = mix_lds(Vs[0]) + wave * 1024;
    auto fetch = [&](int s, int into) {
        const int key0 = key_of(s), left = (s < nsink ? range.sink_end : range.hi) - key0;
        kt.fetch(Kb + (size_t)key0 * p.k.l, left, p.k.l, klds + into * (AK * DW * 4));
        vt.fetch(Vb + (size_t)key0 * p.v.l, left, p.v.l, vlds + into * (AK * DW * 4));
    };

    v16f o[DC];
#pragma unroll
    for (int b = 0; b < DC; b++) o[b] = (v16f)(0.0f);
    // Scores are formed relative to a reference: the accumulators start at its negative, so the exponentials need no
    // subtraction.  It starts at the first scores' maximum (until then it is 0 and `raise` lets any score through) and is
    // raised only when some score exceeds it by 2^LAG -- any reference gives the same result after the final division.
    v16f from = (v16f)(0.0f);                               // minus the reference, 16 times
    float raise = LOWEST, l = 0.0f;                         // l: this half's sum

    if (first < last) fetch(first, 0);
    mix_wait();               // also for the loads above: the compiler would wait for them, and the step's transfers, in every step
    __syncthreads();
    auto step = [&](auto bufc, int s) {
        constexpr int buf = decltype(bufc)::value;
        if (s + 1 < last) fetch(s + 1, buf ^ 1);            // nobody reads that buffer during this step
        __builtin_amdgcn_sched_barrier(0);
        const int key0 = key_of(s), limit = s < nsink ? range.sink_end : range.hi, end = min(key0 + AK, limit);
        // a wavefront none of whose queries sees a key of this step has nothing to do
        const bool sees = w0 <= w1 && (s < nsink || (key0 <= w1 && (end - 1 > w0 - p.window || key0 < p.sinks)));
        if (sees) {
            v16f sc[KB];
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                sc[kb] = from;
                mix_rows_product<DW, NG>(sc[kb], Ks[buf] + kb * 32 * DW, qf, r, h);
            }
            // keys behind a query (or behind the last key), and before its window: tested only where some query has them
            if (key0 + AK - 1 > w0 || key0 + AK > limit || !span.full) {
                const int top = min(pos, limit - 1) - key0 - 4 * h;
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (32 * kb + mix_row(v, 0) > top) sc[kb][v] = NEG;
            }
            if (s >= nsink && key0 <= w1 - p.window) {
                const int low = pos - p.window - key0 - 4 * h, sink = p.sinks - key0 - 4 * h;
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (32 * kb + mix_row(v, 0) <= low && 32 * kb + mix_row(v, 0) >= sink) sc[kb][v] = NEG;
            }
            float mt = sc[0][0];
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int v = (kb == 0); v < 16; v++) mt = fmaxf(mt, sc[kb][v]);
            const MixHalves both = mix_halves(mt);
            mt = fmaxf(both.a, both.b);
            if (__builtin_amdgcn_ballot_w64(mt > raise) != 0) {
                const bool begun = raise != LOWEST;
                const float up = begun ? fmaxf(mt, 0.0f) : (mt == NEG ? 0.0f : mt);
                const float alpha = begun ? __builtin_amdgcn_exp2f(-up) : 0.0f;
                if (mt > raise) raise = (float)LAG;
                l *= alpha;
                from -= up;
#pragma unroll
                for (int kb = 0; kb < KB; kb++) sc[kb] -= up;
#pragma unroll
                for (int b = 0; b < DC; b++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[b][v] *= alpha;
            }
            float sum = 0.0f;
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    sc[kb][v] = __builtin_amdgcn_exp2f(sc[kb][v]);
                    sum += sc[kb][v];
                }
            l += sum;
#pragma unroll
            for (int kb = 0; kb < KB; kb++) mix_columns_product<DW, DC, false>(o, Vs[buf] + kb * 32 * DW, sc[kb], vcols);
        }
        mix_wait();
        __syncthreads();
    };
    for (int s = first; s < last; s += 2) {                 // the buffer is a constant in each copy of the step
        step(std::integral_constant<int, 0>{}, s);
        if (s + 1 < last) step(std::integral_constant<int, 1>{}, s + 1);
    }

    const MixHalves sums = mix_halves(l);
    l = sums.a + sums.b;
    const float m = raise == LOWEST ? NEG : -from[0];
    if (!row.exists) return;
    if (p.parts == 1) {
        mix_store_row<DC>(p.Y + job.n * p.y.n + row.hd * p.y.h + (size_t)row.i * p.y.l, o, l == 0.0f ? 0.0f : 1.0f / l, p.dv4, h);
        if (p.Lse != nullptr && h == 0) p.Lse[stat] = window_lse(m, l);
    } else {
        mix_store_row<DC>(window_part_o(p, cutting, part.slot, wrow + r - row0), o, 1.0f, p.dv4, h);
        if (h == 0) window_part_ml(p, cutting, part.slot, wrow + r - row0) = make_float2(m, l);
    }
}

// ---------------------------------------------------------------- few queries
// A wavefront's 16 rows are (query, head of the group) pairs: row = query * group + head.  Lane (c, k4) = (lane & 15,
// lane >> 4).  S^T = K.Q^T: lane holds 16 bytes of key c per 16 floats of the head dimension, at 4 * k4; MFMA step u of that
// chunk multiplies d = 16s + 4*k4 + u.  Result register v of lane (c, k4) is key 4*k4 + v, row c: the B operand of step v of
// Y^T = V^T.P^T, whose A operand is key 4*k4 + v.  A lane loads 16 bytes of that key at 64*e + 4*c; its float u belongs to
// the 16 outputs 64e + 4*(0..15) + u, so the four floats feed four blocks.
template <int DE, bool NT>   // head dimension in 64s; keys and values read non-temporally
__global__ __launch_bounds__(NTHREADS, 2) void window_rows(const WindowParams p) {
    constexpr int NS = DE * 4;
    constexpr WindowCutting cutting = ROWS_CUTTING;
    __shared__ __attribute__((aligned(16))) float So[4][16][DE * 64 + 4];
    __shared__ float Sm[4][16], Sl[4][16];

    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, k4 = lane >> 4;
    const WindowPart part = window_part(p, cutting, blockIdx.x);
    if (part.none) return;
    const WindowJob job = part.job;
    const WindowLens len = window_lens(p, job.n);
    const int group = p.head / p.kv_head, rows = p.QL * group, off = len.vl - len.ql;
    const int row0 = job.qt * 16;
    const WindowRow row = window_row(p, job, row0 + c, group, len.ql);
    const bool live = row.live;
    const int pos = live ? row.i + off : -1;

    const WindowSpan all = window_span(row0, 16, group, len.ql, off);
    const WindowRange range = window_range(p, all.first, all.last, all.first <= all.last, len.vl);
    const int nsink = (range.sink_end + 15) / 16, nwin = (max(range.hi - range.low, 0) + 15) / 16;
    const int first = mix_uniform((int)((long long)(nsink + nwin) * job.part / part.parts));
    const int last = mix_uniform((int)((long long)(nsink + nwin) * (job.part + 1) / part.parts));

    const float* qrow = p.Q + job.n * p.q.n + row.hd * p.q.h + (size_t)row.i * p.q.l;
    v4f qf[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const int d = 16 * s + 4 * k4;
        qf[s] = (live && d < p.dk4) ? *(const v4f*)(qrow + d) * p.c : (v4f)(0.0f);
    }

    const float* Kb = p.K + job.n * p.k.n + job.kvh * p.k.h;
    const float* Vb = p.V + job.n * p.v.n + job.kvh * p.v.h;
    int koff[NS], voff[4 * DE];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const int d = 16 * s + 4 * k4;
        koff[s] = d < p.dk4 ? (c * p.k.l + d) * 4 : OOB_OFFSET;
    }
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
        for (int e = 0; e < DE; e++) {
            const int d = 64 * e + 4 * c;
            voff[v * DE + e] = d < p.dv4 ? ((4 * k4 + v) * p.v.l + d) * 4 : OOB_OFFSET;
        }
    v4f kr[NS], vr[4 * DE];
    auto fetch = [&](int s) {
        const int key0 = s < nsink ? s * 16 : range.low + (s - nsink) * 16;
        const int left = min((s < nsink ? range.sink_end : range.hi) - key0, 16);
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(Kb + (size_t)key0 * p.k.l), 0, left * p.k.l * 4, RSRC_FLAGS);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(Vb + (size_t)key0 * p.v.l), 0, left * p.v.l * 4, RSRC_FLAGS);
#pragma unroll
        for (int s2 = 0; s2 < NS; s2++) kr[s2] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rk, koff[s2], 0, NT ? 2 : 0));
#pragma unroll
        for (int s2 = 0; s2 < 4 * DE; s2++) vr[s2] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rv, voff[s2], 0, NT ? 2 : 0));
    };

    v4f o[DE][4];
#pragma unroll
    for (int e = 0; e < DE; e++)
#pragma unroll
        for (int u = 0; u < 4; u++) o[e][u] = (v4f)(0.0f);
    float m = NEG, l = 0.0f;

    const int uwave = __builtin_amdgcn_readfirstlane(wave);
    if (first + uwave < last) fetch(first + uwave);
    for (int s = first + uwave; s < last; s += 4) {
        const int key0 = s < nsink ? s * 16 : range.low + (s - nsink) * 16;
        const int limit = s < nsink ? range.sink_end : range.hi;
        v4f kc[NS], vc[4 * DE];
#pragma unroll
        for (int s2 = 0; s2 < NS; s2++) kc[s2] = kr[s2];
#pragma unroll
        for (int s2 = 0; s2 < 4 * DE; s2++) vc[s2] = vr[s2];
        if (s + 4 < last) fetch(s + 4);
        v4f sc = (v4f)(0.0f), odd = (v4f)(0.0f);                // two sums: half the roundings in a row, half the wait
#pragma unroll
        for (int s2 = 0; s2 < NS; s2++)
#pragma unroll
            for (int u = 0; u < 4; u += 2) {
                sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kc[s2][u], qf[s2][u], sc, 0, 0, 0);
                odd = __builtin_amdgcn_mfma_f32_16x16x4f32(kc[s2][u + 1], qf[s2][u + 1], odd, 0, 0, 0);
            }
        sc += odd;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int j = key0 + 4 * k4 + v;
            if (!(j < limit && window_sees(p, pos, j))) sc[v] = NEG;
        }
        float mt = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        if (__builtin_amdgcn_ballot_w64(mt > m + (float)LAG) != 0) {
            const float m_new = fmaxf(m, mt);
            const float alpha = m == NEG ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int e = 0; e < DE; e++)
#pragma unroll
                for (int u = 0; u < 4; u++) o[e][u] *= alpha;
        }
        const float ref = fmaxf(m, LOWEST);
#pragma unroll
        for (int v = 0; v < 4; v++) {
            sc[v] = __builtin_amdgcn_exp2f(sc[v] - ref);
            l += sc[v];
        }
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int e = 0; e < DE; e++)
#pragma unroll
                for (int u = 0; u < 4; u++) o[e][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(vc[v * DE + e][u], sc[v], o[e][u], 0, 0, 0);
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // ---- the four wavefronts' parts of the keys, added through LDS; register w of block (e, u) is d = 64e + 16*k4 + 4w + u ----
#pragma unroll
    for (int e = 0; e < DE; e++)
#pragma unroll
        for (int w = 0; w < 4; w++)
            *(v4f*)&So[wave][c][64 * e + 16 * k4 + 4 * w] = (v4f){o[e][0][w], o[e][1][w], o[e][2][w], o[e][3][w]};
    if (k4 == 0) { Sm[wave][c] = m; Sl[wave][c] = l; }
    __syncthreads();
    for (int x = t; x < 16 * (p.dv4 / 4); x += NTHREADS) {
        const int rr = x / (p.dv4 / 4), d = 4 * (x - rr * (p.dv4 / 4));
        if (row0 + rr >= rows) break;
        const float M = fmaxf(fmaxf(Sm[0][rr], Sm[1][rr]), fmaxf(Sm[2][rr], Sm[3][rr]));
        float L = 0.0f;
        v4f y = (v4f)(0.0f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = Sm[w][rr] == NEG ? 0.0f : __builtin_amdgcn_exp2f(Sm[w][rr] - M);
            L += Sl[w][rr] * f;
            y += *(const v4f*)&So[w][rr][d] * f;
        }
        const int qi = (row0 + rr) / group, qh = job.kvh * group + (row0 + rr - qi * group);
        const size_t stat = ((size_t)job.n * p.head + qh) * p.QL + qi;
        if (p.parts == 1) {
            *(v4f*)(p.Y + job.n * p.y.n + qh * p.y.h + (size_t)qi * p.y.l + d) = L == 0.0f ? (v4f)(0.0f) : y * (1.0f / L);
            if (p.Lse != nullptr && d == 0) p.Lse[stat] = window_lse(M, L);
        } else {
            *(v4f*)(window_part_o(p, cutting, part.slot, rr) + d) = y;
            if (d == 0) window_part_ml(p, cutting, part.slot, rr) = make_float2(M, L);
        }
    }
}

// ---------------------------------------------------------------- the parts of a row, added in order
// `wide` threads (16 or 32) for a row's columns, `across` of such groups (a power of two up to 8) next to each other for its
// parts: a thread adds every across-th part, LDS joins the rest.  With few rows and many parts one thread for all of them
// would read one after the other: 64 parts of 32 rows in 22.3 us, so in 4.7.
__global__ __launch_bounds__(NTHREADS) void window_join(const WindowParams p, const WindowCutting c, int wide, int across) {
    __shared__ __attribute__((aligned(16))) v4f Sy[NTHREADS];
    __shared__ float2 Sml[NTHREADS / 16];
    const int t = threadIdx.x, slot = t / wide, sub = slot & (across - 1), d = 4 * (t & (wide - 1));
    const long long stat = (long long)blockIdx.x * (NTHREADS / wide / across) + slot / across;
    const bool mine = stat < (long long)p.N * p.head * p.QL && d < p.dv4;
    const long long nh = stat / p.QL;
    const int n = (int)(nh / p.head), hd = (int)(nh - (long long)n * p.head), i = (int)(stat - nh * p.QL);
    float M = NEG, L = 0.0f;
    v4f y = (v4f)(0.0f);
    if (mine) {
        const int group = p.head / p.kv_head, kvh = hd / group, row = i * group + hd - kvh * group, tile = row / c.per;
        const int pair = (p.qtiles - 1 - tile) * p.N + n, in = row - tile * c.per;
        const int2 deal = c.deal ? window_part_deal(p, c, pair) : make_int2(pair * p.parts, p.parts);
        const int parts = deal.y, slot = kvh * p.N * p.qtiles * p.parts + deal.x;
#pragma unroll 4
        for (int s = sub; s < parts; s += across) M = fmaxf(M, window_part_ml(p, c, slot + s, in).x);
#pragma unroll 4
        for (int s = sub; s < parts; s += across) {
            const float2 ml = window_part_ml(p, c, slot + s, in);
            const float f = ml.x == NEG ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
            L += ml.y * f;
            y += *(const v4f*)(window_part_o(p, c, slot + s, in) + d) * f;
        }
    }
    if (across > 1) {
        Sy[t] = y;
        if (d == 0) Sml[slot] = make_float2(M, L);
        __syncthreads();
        if (sub != 0) return;
        for (int s = 1; s < across; s++) M = fmaxf(M, Sml[slot + s].x);
        L = 0.0f;
        y = (v4f)(0.0f);
        for (int s = 0; s < across; s++) {
            const float2 ml = Sml[slot + s];
            const float f = ml.x == NEG ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
            L += ml.y * f;
            y += Sy[t + s * wide] * f;
        }
    }
    if (!mine) return;
    *(v4f*)(p.Y + n * p.y.n + hd * p.y.h + (size_t)i * p.y.l + d) = L == 0.0f ? (v4f)(0.0f) : y * (1.0f / L);
    if (p.Lse != nullptr && d == 0) p.Lse[stat] = window_lse(M, L);
}

// ---------------------------------------------------------------- host side
constexpr long long JOIN_ROWS = 1024;    // rows from which a thread of window_join takes all parts (500 x 8 rows: 63 us, else 67)
// Rows of a key / value head up to which window_rows takes the call.  64 rows on 16 x 8192 keys of 8 heads of 128 under a window
// of 1024: 51 us (window_tiles 79), on 8 x 4096 all: 97 (136); but 72 rows on 2 x 4096: 52 (49), 96 rows: 64 (51).
constexpr int ROWS_MAX = 64;

struct WindowPlan { bool rows; int qtiles, parts, per; };

// One decision for the launch and for the size of the caller's buffer: from the sizes alone.  The keys are cut where there are
// fewer workgroups than wanted; for tiles of 128 rows under a window, which differ little, fewer than half of them.  (Tiles that
// see everything before them: 256 tiles of 64 columns 78 -> 65 us, 320 of 128: 164 -> 123; cut for twice as many: 131.)
// A part of window_rows is worth its launch of window_join from 8 steps on, if there are 24 to cut: one token on 1024 keys of 4
// heads of 64 in 10.0 us (cuts of 16: 11.2), but on 256 keys 7.9 whole and 9.4 cut.  More parts than compute units gain nothing
// there (16384 keys of 8 heads of 128: 29 us, with twice as many 33).
// At most 64 parts, which bounds the work buffer: one token on 65536 keys of one head of 128 takes 33 us (32 parts: 54; 256, as
// many as compute units, would take 26, and 128 queries of one head there 52 instead of 138); on 4 heads, which fill the units, 51.
WindowPlan window_plan(int N, int head, int kv_head, int QL, int VL, int window, int sinks) {
    WindowPlan x;
    const long long group = head / kv_head, rows = QL * group;
    x.rows = rows <= ROWS_MAX;
    const long long per = x.per = x.rows ? 16 : AQ;
    x.qtiles = (int)((rows + per - 1) / per);
    const long long base = (long long)N * kv_head * x.qtiles;
    const long long reach = window == 0 ? VL : (long long)window + sinks + (per + group - 1) / group;
    const long long steps = ((reach < VL ? reach : VL) + (x.rows ? 15 : 31)) / (x.rows ? 16 : 32);
    const WindowCutting c = x.rows ? ROWS_CUTTING : tile_cutting(32, false);
    const long long want = c.want, least = x.rows && steps < 24 ? 24 : c.least;
    long long parts = base >= (!x.rows && reach < VL ? want / 2 : want) ? 1 : (want + base - 1) / base;
    if (parts > steps / least) parts = steps / least;
    x.parts = (int)(parts < 1 ? 1 : parts > 64 ? 64 : parts);
    return x;
}

long long window_workgroups(const WindowPlan& x, int N, int kv_head) { return (long long)N * kv_head * x.qtiles * x.parts; }
// the join's: rows a workgroup, threads side by side for a row's parts
struct WindowJoin { int wide, across; long long workgroups; };
WindowJoin window_join_plan(const WindowPlan& x, int N, int head, int QL, int dv4) {
    const long long rows = (long long)N * head * QL;
    WindowJoin j;
    j.wide = dv4 <= 64 ? 16 : 32;
    j.across = rows >= JOIN_ROWS ? 1 : x.parts >= 8 ? 8 : x.parts >= 4 ? 4 : 2;
    const int per = NTHREADS / j.wide / j.across;
    j.workgroups = x.parts == 1 ? 0 : (rows + per - 1) / per;
    return j;
}
bool window_launches_fit(const WindowPlan& x, int N, int head, int kv_head, int QL, int dv4) {
    return mix_launch_fits(window_workgroups(x, N, kv_head), NTHREADS) &&
           mix_launch_fits(window_join_plan(x, N, head, QL, dv4).workgroups, NTHREADS);
}

long long window_buffer(const WindowPlan& x, int N, int kv_head, int dv4) {
    return x.parts == 1 ? 0 : (long long)N * kv_head * x.qtiles * x.parts * x.per * (dv4 + 2) * 4 + (long long)N * x.qtiles * 8;
}

}  // namespace

bool window_arguments_ok(int N, int head, int kv_head, int QL, int VL, int dk4, int dv4, int window, int sinks) {
    if (N <= 0 || head <= 0 || kv_head <= 0 || head % kv_head != 0 || QL <= 0 || VL <= 0 || dk4 <= 0 || dv4 <= 0 || (dk4 & 3) ||
        (dv4 & 3) || dk4 > 128 || dv4 > 128 || window < 0 || sinks < 0)
        return false;
    // positions and rows are 32-bit, a tile's offsets 32-bit bytes, key tiles over all sequences and rows over 16 31 bits.  (What a
    // launch takes is asked of the forward pass's and the gradient's own plans.)
    const long long row = (long long)head * (dk4 > dv4 ? dk4 : dv4);
    return (long long)QL + VL < 0x3fffff00LL && row * AQ * 4 < 0x7ffffff0LL && (long long)QL * (head / kv_head) < 0x7fffff00LL &&
           (long long)N * kv_head * ((VL + 127LL) / 128) < 0x7fffffffLL &&
           (long long)N * head * ((QL + 15LL) / 16) * 64 < 0x7fffffffLL;
}

}  // namespace dragon

using namespace dragon;

extern "C" {

void dragon_window_deal_bounds(double all, int32_t slots, int32_t pairs, int32_t least, int32_t* lo, int32_t* hi) {
    const WindowDealBounds x = window_deal_bounds(all, slots, pairs, least);
    *lo = x.lo;
    *hi = x.hi;
}

int64_t dragon_Cuda_attention_window_bufsize(int32_t N, int32_t head, int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4,
                                             int32_t dV4, int32_t window, int32_t sinks) {
    if (!window_arguments_ok(N, head, kv_head, QL, VL, dK4, dV4, window, sinks)) return -1;
    const WindowPlan plan = window_plan(N, head, kv_head, QL, VL, window, sinks);
    return window_launches_fit(plan, N, head, kv_head, QL, dV4) ? window_buffer(plan, N, kv_head, dV4) : -1;
}

int dragon_Cuda_attention_window_forward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV, int64_t dY,
                                         int64_t dLse, int64_t dQLens, int64_t dVLens, int64_t dBuf, int64_t buf_size, int32_t N,
                                         int32_t head, int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4, int32_t dV4,
                                         int32_t head_inner, float scale, int32_t window, int32_t sinks) {
    if (streams == nullptr || length < 1 || length > 10) return hipErrorInvalidValue;
    if (dQ == 0 || dK == 0 || dV == 0 || dY == 0 || !mix_aligned16(dQ) || !mix_aligned16(dK) || !mix_aligned16(dV) ||
        !mix_aligned16(dY) || (dLse & 3) || (dQLens & 3) || (dVLens & 3))
        return hipErrorInvalidValue;
    if (!window_arguments_ok(N, head, kv_head, QL, VL, dK4, dV4, window, sinks) || !(scale - scale == 0.0f))
        return hipErrorInvalidValue;
    const WindowPlan plan = window_plan(N, head, kv_head, QL, VL, window, sinks);
    if (!window_launches_fit(plan, N, head, kv_head, QL, dV4)) return hipErrorInvalidValue;
    const long long need = window_buffer(plan, N, kv_head, dV4);
    if (need > 0 && (dBuf == 0 || !mix_aligned16(dBuf) || buf_size < need)) return hipErrorInvalidValue;

    WindowParams p;
    p.Q = (const float*)(intptr_t)dQ; p.K = (const float*)(intptr_t)dK; p.V = (const float*)(intptr_t)dV;
    p.Y = (float*)(intptr_t)dY; p.Lse = (float*)(intptr_t)dLse;
    p.QLens = (const int*)(intptr_t)dQLens; p.VLens = (const int*)(intptr_t)dVLens;
    p.N = N; p.head = head; p.kv_head = kv_head; p.QL = QL; p.VL = VL; p.dk4 = dK4; p.dv4 = dV4;
    p.q = mix_layout(head_inner, head, QL, dK4); p.y = mix_layout(head_inner, head, QL, dV4);
    p.k = mix_layout(head_inner, kv_head, VL, dK4); p.v = mix_layout(head_inner, kv_head, VL, dV4);
    p.window = window == 0 || window > QL + VL ? QL + VL : window;
    p.sinks = sinks;
    p.c = scale * MIX_LOG2E;
    p.qtiles = plan.qtiles; p.parts = plan.parts;
    p.part = need > 0 ? (float*)(intptr_t)dBuf : nullptr;
    split_ledger_touch(p.Y, (size_t)N * head * QL * dV4 * 4);
    if (p.Lse != nullptr) split_ledger_touch(p.Lse, (size_t)N * head * QL * 4);
    if (p.part != nullptr) split_ledger_touch(p.part, (size_t)need);

    hipStream_t s = (hipStream_t)(intptr_t)streams[0];
    const int dmax = dK4 > dV4 ? dK4 : dV4;
    const dim3 block(NTHREADS);
    const dim3 grid((unsigned)window_workgroups(plan, N, kv_head));
    const bool deal = !plan.rows && plan.parts > 1 && (p.QLens != nullptr || p.VLens != nullptr);
    if (plan.rows) {
        // keys and values that are read once and do not fit the Infinity Cache pass it by (stream_policy.h has the border):
        // 65536 keys of 8 heads of 128 in 84 us instead of 96, but 16 x 2048 in 66 instead of 50
        const long long reach = window == 0 || window > VL ? VL : (long long)window + sinks;
        const bool nt = plan.qtiles == 1 && (long long)N * kv_head * (reach < VL ? reach : VL) * (dK4 + dV4) * 4 >= STREAM_NT_BYTES;
        if (dmax <= 64) {
            if (nt) hipLaunchKernelGGL((window_rows<1, true>), grid, block, 0, s, p);
            else hipLaunchKernelGGL((window_rows<1, false>), grid, block, 0, s, p);
        } else {
            if (nt) hipLaunchKernelGGL((window_rows<2, true>), grid, block, 0, s, p);
            else hipLaunchKernelGGL((window_rows<2, false>), grid, block, 0, s, p);
        }
    } else {
#define TILES(...)                                                                                        \
    do {                                                                                                  \
        if (deal) hipLaunchKernelGGL((window_tiles<__VA_ARGS__, true>), grid, block, 0, s, p);            \
        else hipLaunchKernelGGL((window_tiles<__VA_ARGS__, false>), grid, block, 0, s, p);                \
    } while (0)
        switch ((dmax + 31) / 32) {
            case 1: TILES(1, 1, 2); break;
            case 2: TILES(2, 2, 1); break;
            case 3: TILES(4, 3, 1); break;
            default: TILES(4, 4, 1); break;
        }
#undef TILES
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && plan.parts > 1) {
        const WindowJoin join = window_join_plan(plan, N, head, QL, dV4);
        const WindowCutting cutting = plan.rows ? ROWS_CUTTING : tile_cutting(32, deal);     // (the keys of a step are not asked for)
        hipLaunchKernelGGL(window_join, dim3((unsigned)join.workgroups), block, 0, s, p, cutting, join.wide, join.across);
        e = hipGetLastError();
    }
    return e;
}

}  // extern "C"
