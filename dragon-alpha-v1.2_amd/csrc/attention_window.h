// What the forward and the gradient of windowed attention share: parameters, who sees whom, how the work is dealt.
#pragma once
#include "token_mixer.h"

namespace dragon {
namespace {

struct WindowParams {
    const float* Q; const float* K; const float* V; float* Y; float* Lse;
    const int* QLens; const int* VLens;      // valid queries / keys per sequence; null: all of them
    int N, head, kv_head, QL, VL, dk4, dv4;
    MixLayout q, k, v, y;
    int window, sinks;                       // window >= 1 (all keys: the host passes more than there are positions)
    float c;                                 // scale * log2(e): the exponentials are base 2
    int qtiles, parts;                       // workgroups along the rows; cuts of the keys
    float* part;                             // parts > 1: the parts' results (attention_window.hip, attention_window_grad.hip)
};

// (n is the same for the whole wavefront wherever this is called but in window_delta, which has lengths of its own)
struct WindowLens { int ql, vl; };
__device__ __forceinline__ WindowLens window_lens(const WindowParams& p, int n) {
    WindowLens x;
    x.ql = p.QLens ? min(max(mix_uniform(p.QLens[n]), 0), p.QL) : p.QL;
    x.vl = p.VLens ? min(max(mix_uniform(p.VLens[n]), 0), p.VL) : p.VL;
    return x;
}

__device__ __forceinline__ bool window_sees(const WindowParams& p, int pos, int j) {
    const int back = pos - j;
    return back >= 0 && (back < p.window || j < p.sinks);
}

// the keys that positions p0 .. p1 see: [0, sink_end) and [low, hi)
struct WindowRange { int sink_end, low, hi; };
__device__ __forceinline__ WindowRange window_range(const WindowParams& p, int p0, int p1, bool any, int vl) {
    WindowRange x;
    x.hi = any ? max(min(vl, p1 + 1), 0) : 0;
    x.low = any ? min(max(p0 - p.window + 1, 0), x.hi) : 0;
    x.sink_end = min(p.sinks, x.low);
    return x;
}

// log sum exp from a maximum in units of log2 and the sum over it
__device__ __forceinline__ float window_lse(float m, float l) {
    return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * MIX_LN2;   // logf is base 2
}

// The rows of a tile are (query, query head) pairs of one key / value head, row = query * group + head: heads that share their
// keys share the tiles, and a tile spans as few positions as can be -- 128 / group of them, so that under a window it has
// that much less to walk over than its rows see.  Workgroups of one key / value head follow each other at a distance of
// N * kv_head; where that is a multiple of the 8 XCDs (to which workgroups are dealt in turn) a head's keys are read by one
// XCD's L2 alone.  The tiles at the end of the sequence, which see the most keys, start first.
struct WindowJob { int n, kvh, qt, part; };
__device__ __forceinline__ WindowJob window_job(const WindowParams& p, int id) {
    const int nkv = p.N * p.kv_head;
    WindowJob x;
    const int a = mix_uniform(id / nkv), kv = id - a * nkv;
    const int qx = mix_uniform(a / p.parts);
    x.part = a - qx * p.parts;
    x.qt = p.qtiles - 1 - qx;
    x.n = mix_uniform(kv / p.kv_head);
    x.kvh = kv - x.n * p.kv_head;
    return x;
}

// rows [row0, row0 + count) of a key / value head: the positions of the first and of the last that exist (first > last: none),
// and whether all count exist
struct WindowSpan { int first, last; bool full; };
__device__ __forceinline__ WindowSpan window_span(int row0, int count, int group, int ql, int off) {
    WindowSpan x;
    const int rows = ql * group, end = min(row0 + count, rows);
    x.first = mix_uniform(row0 / group) + off;
    x.last = end > row0 ? mix_uniform((end - 1) / group) + off : x.first - 1;
    x.full = row0 + count <= rows;
    return x;
}
// a lane's row: its query, its head; dead behind the sequence's queries
struct WindowRow { int i, hd; bool exists, live; };
__device__ __forceinline__ WindowRow window_row(const WindowParams& p, const WindowJob& job, int row, int group, int ql) {
    WindowRow x;
    const int i = row / group;
    x.exists = i < p.QL;
    x.live = i < ql;
    x.i = min(i, p.QL - 1);
    x.hd = job.kvh * group + (row - i * group);
    return x;
}

}  // namespace
}  // namespace dragon
