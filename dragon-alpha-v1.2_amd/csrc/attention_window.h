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
    int qtiles, parts;                       // workgroups along the queries; cuts of the keys
    float* part;                             // parts > 1: the parts' outputs, behind them their (maximum, sum)

    __device__ __forceinline__ float* part_o(size_t row, int s) const { return part + (row * parts + s) * dv4; }
    __device__ __forceinline__ float2& part_ml(size_t row, int s) const {
        return ((float2*)(part + (size_t)N * head * QL * parts * dv4))[row * parts + s];
    }
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

// Workgroups of one key / value head follow each other at a distance of N * kv_head, so where that is a multiple of the 8
// XCDs (to which workgroups are dealt in turn) a head's keys are read by one XCD's L2 alone; and the tiles at the end of the
// sequence, which see the most keys, start first.
struct WindowJob { int n, kvh, hd, qt, part; };
__device__ __forceinline__ WindowJob window_job(const WindowParams& p, int id) {
    const int nkv = p.N * p.kv_head, group = p.head / p.kv_head;
    WindowJob x;
    const int a = mix_uniform(id / nkv), kv = id - a * nkv;
    const int b = mix_uniform(a / group), g = a - b * group;
    const int qx = mix_uniform(b / p.parts);
    x.part = b - qx * p.parts;
    x.qt = p.qtiles - 1 - qx;
    x.n = mix_uniform(kv / p.kv_head);
    x.kvh = kv - x.n * p.kv_head;
    x.hd = x.kvh * group + g;
    return x;
}
__device__ __forceinline__ WindowJob window_row_job(const WindowParams& p, int id) {
    const int nkv = p.N * p.kv_head;
    WindowJob x;
    const int a = mix_uniform(id / nkv), kv = id - a * nkv;
    x.qt = mix_uniform(a / p.parts);
    x.part = a - x.qt * p.parts;
    x.n = mix_uniform(kv / p.kv_head);
    x.kvh = kv - x.n * p.kv_head;
    x.hd = 0;
    return x;
}

}  // namespace
}  // namespace dragon
