// Linear attention with a decay for each head: a state S[dk, dv] per (image, head) that forgets by a constant factor a token,
//     S_t = e^g S_{t-1} + K[t]^T V[t],     Y[t] = scale * Q[t] S_t            (g <= 0, one per head)
// and its gradient.
//
// Few tokens (decay_steps): the recurrence itself, the state in registers; bound by reading and writing the states: a token of
// 256 x 32 states of 128 x 128 in 193 us, 5.6 TB/s; from the third token or so on by the vector instructions, four an element
// and token (64 x 32 states: 44 us for one token, 59 for four, 108 for twelve).
// Many tokens (decay_walk): 32 at a time.  With S the state before them and t a token's place among them,
//     Y[t] = scale * (e^{g(t+1)} Q[t] S  +  sum_{j <= t} e^{g(t-j)} <Q[t], K[j]> V[j]),    S' = e^{32g} S + sum_j e^{g(31-j)} K[j]^T V[j]
// A workgroup walks along a sequence with the state in its registers, a wavefront for each 32 columns of V.  Where there are
// fewer (image, head) pairs than the chip takes workgroups the sequence is cut into segments that walk at the same time:
// decay_states forms each segment's own sum, decay_scan runs over them and leaves the state that each begins with.
// Bound by the FP32 matrix pipe: 2.5 products of [dk, dv] size a token, and one more where there are segments.  16 heads of 128
// and 32768 tokens: the states 146 to 157 us (113 TFLOP/s), the scan 13, the walk 380 to 420 (106), the pipes busy for 74 % of both; the
// rest of the walk goes to vector instructions (powers, decay of the state) and to two barriers for 32 tokens.
//
// The gradient is the same walk with other operands (G = gradient of Y, sums over j >= t in the last two, from the end):
//     dQ[t] = scale sum e^{g(t-j)} <G[t], V[j]> K[j] + ...  S^T           the states of the forward pass again
//     dK[t] = scale sum e^{g(j-t)} <V[t], G[j]> Q[j] + ...  R^T           R: the same sum from the sequence's end,
//     dV[t] = scale sum e^{g(j-t)} <K[t], Q[j]> G[j] + ...  R             over Q^T G, starting with the gradient of the last state
// so decay_walk takes its operands x, y, z by name, a direction, and the beginning state either way round.
//
// Every power e^{g n} is computed as such (n >= 0: it cannot overflow), never as a quotient of two powers.  States, sums and
// powers are FP32.  An exponent is g times log2(e), rounded, times n, rounded: with the constant's own error up to 2.2 |g n| 2^-24
// in a power, beside the last bit of exp2, and a power of decay_states is the product of two.  Those errors meet a token's share
// once; the factors that meet the state again and again are another matter (decay_slow).
#include "token_mixer.h"
#include "runtime_internal.h"
#include "stream_policy.h"
#include "../../include/dragon_hip_gemm.h"

namespace dragon {
namespace {

struct DecayWalk {
    const float* x; const float* y; const float* z; float* out;   // [L, xd], [L, xd], [L, zd], [L, zd] per (image, head)
    MixLayout lx, lz;                                             // of x and y, of z and out
    const float* g; const int* lens;
    int head, L, xd, zd;
    int segment, segments;     // tokens of a segment, a multiple of 32
    int back;                  // sums over j >= t instead of j <= t
    float near_scale, far_scale, add_scale;   // factors on the sum inside 32 tokens, on the state's share, on what enters the state
    const float* state;        // what each segment begins with (back: at its end), [image, head, segment]; null: zeros
    float* last;               // one segment: the state at the other end; null: nobody wants it
    int nh;                    // image-head pairs
};

__device__ __forceinline__ float decay_log2(float g) {
    // not below -1e30: 0 * g has to be 0 where the head forgets at once (g = -infinity); NaN stays NaN
    const float g2 = g * MIX_LOG2E;
    return g2 < -1.0e30f ? -1.0e30f : g2;
}
__device__ __forceinline__ float decay_pow(float g2, int n) { return __builtin_amdgcn_exp2f(g2 * (float)n); }
// What n >= 1 tokens leave of a state.  The same factor meets it again and again, so an error of the factor adds up in one
// direction: rounded to FP32, a factor near 1 is off by up to 2^-25 every time (a state of a head that remembers them was off
// by 6e-5 after 1800 factors).  So a head that keeps at least half takes (1 - e^{gn}) S off instead, a difference with a small error of
// its own, and only the rounding of S itself is left, which goes up as often as down: 7e-8 there.  (Below a half the difference
// would cancel; such a head forgets its errors too.)
__device__ __forceinline__ bool decay_slow(float g, int n) { return fabsf(g * (float)n) < MIX_LN2; }
// e^{gn} - 1 of such a head: Taylor's series to x^10, what is left out is below 2^-26 of it
__device__ __forceinline__ float decay_less(float g, int n) {
    const float x = g * (float)n;
    float s = 1.0f / 3628800.0f;
    s = __builtin_fmaf(s, x, 1.0f / 362880.0f);
    s = __builtin_fmaf(s, x, 1.0f / 40320.0f);
    s = __builtin_fmaf(s, x, 1.0f / 5040.0f);
    s = __builtin_fmaf(s, x, 1.0f / 720.0f);
    s = __builtin_fmaf(s, x, 1.0f / 120.0f);
    s = __builtin_fmaf(s, x, 1.0f / 24.0f);
    s = __builtin_fmaf(s, x, 1.0f / 6.0f);
    s = __builtin_fmaf(s, x, 0.5f);
    return __builtin_fmaf(x * x, s, x);
}
// for both kinds of heads in one expression: S <- keep S + f S, keep 1 or 0
struct DecayFactor { float keep, f; };
__device__ __forceinline__ DecayFactor decay_factor(float g, int n) {
    const bool slow = decay_slow(g, n);
    const float less = decay_less(g, n), power = decay_pow(decay_log2(g), n);
    return {slow ? 1.0f : 0.0f, slow ? less : power};
}
__device__ __forceinline__ int decay_len(const int* lens, int n, int L) { return lens ? min(max(lens[n], 0), L) : L; }

// ---------------------------------------------------------------- along the sequence
// Wavefront b of a workgroup owns 32 columns of the state and of the output (as result columns' rows: out^T[32][token]).
//   scores   every wavefront a part of the head dimension; the parts are added through LDS
//   x . S    out^T[column][token] += S^T . x^T: the state's registers are the A operand as they stand
//   near     out^T[column][token] += z^T . scores
//   S'       S^T... [row][column] = decayed + y^T . z, the result layout that x . S takes
// XB: 32-wide blocks of x's width in LDS (1, 2, 4), ZB: of z's, one wavefront each.  ST: the beginning state lies [zd][xd].
// Two workgroups share a compute unit (80 KiB of LDS each at widths of 128).  Two barriers for 32 tokens: behind the first the
// scores and z are there and x is free, behind the second z is free and the next x and y are there; y has two buffers.
template <int XB, int ZB, bool ST>
__global__ __launch_bounds__(64 * ZB, XB == 4 && ZB < 3 ? 1 : 2) void decay_walk(const DecayWalk p) {
    constexpr int XW = XB * 32, ZW = (ZB == 3 ? 4 : ZB) * 32, NG = XB * 4, SHARE = (NG + ZB - 1) / ZB;
    __shared__ __attribute__((aligned(1024))) float Xs[32 * XW];
    __shared__ __attribute__((aligned(1024))) float Ys[2][32 * XW];
    __shared__ __attribute__((aligned(1024))) float Zs[32 * ZW];
    __shared__ __attribute__((aligned(16))) float Ps[ZB][1024];
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const int lid = xcd_contiguous_id(blockIdx.x, gridDim.x);   // one XCD works on all heads of the same tokens, which lie side by side
    const int segment = mix_uniform(lid / p.nh), nh = lid - segment * p.nh;
    const int n = mix_uniform(nh / p.head), hd = nh - n * p.head;
    const int len = mix_uniform(decay_len(p.lens, n, p.L));
    const int from = segment * p.segment, end = min(from + p.segment, p.L), to = max(min(end, len), from);
    const float g = p.g[hd], g2 = decay_log2(g);
    const int col = 32 * wave + r;                              // this lane's column of the state
    const float* const xb = p.x + n * p.lx.n + hd * p.lx.h;
    const float* const yb = p.y + n * p.lx.n + hd * p.lx.h;
    const float* const zb = p.z + n * p.lz.n + hd * p.lz.h;
    float* const ob = p.out + n * p.lz.n + hd * p.lz.h + 32 * wave;
    const int mine = p.zd - 32 * wave;                          // floats of a row of `out` from this wavefront's on

    MixTile<XW, 32, true, 64 * ZB> xt;                          // x and y lie alike, z and out too
    MixTile<ZW, 32, false, 64 * ZB> zt;
    MixColumns<XW, true> cols;
    cols.init(r, h);
    xt.init(t, p.lx.l, p.xd);
    zt.init(t, p.lz.l, p.zd);
    const unsigned xlds = mix_lds(Xs) + wave * 1024, ylds = mix_lds(Ys[0]) + wave * 1024, zlds = mix_lds(Zs) + wave * 1024;
    auto fetch_xy = [&](int t0, int into) {
        xt.fetch(xb + (size_t)t0 * p.lx.l, to - t0, p.lx.l, xlds, wave);
        xt.fetch(yb + (size_t)t0 * p.lx.l, to - t0, p.lx.l, ylds + into * (32 * XW * 4), wave);
    };
    auto fetch_z = [&](int t0) { zt.fetch(zb + (size_t)t0 * p.lz.l, to - t0, p.lz.l, zlds, wave); };
    const int chunks = (to - from + 31) / 32;
    auto start = [&](int c) { return from + 32 * (p.back ? chunks - 1 - c : c); };
    if (chunks > 0) {
        fetch_xy(start(0), 0);
        fetch_z(start(0));
    }

    // Everything from here on for either kind of head by itself: a branch around the state in every step costs registers that
    // a state of 128 x 96 does not have (16 x 32 heads of 96, 1024 tokens: 473 us, so 375).
    auto along = [&](auto slowc) {
        constexpr bool SLOW = decltype(slowc)::value;
        // ---- the state that the segment begins with: register v of block k is row 32k + mix_row(v, h), column col ----
        v16f S[XB];
        bool any = p.state != nullptr;                              // the state is not zero all over
#pragma unroll
        for (int k = 0; k < XB; k++) S[k] = (v16f)(0.0f);
        if (any) {
            const float* s0 = p.state + ((size_t)nh * p.segments + segment) * p.xd * p.zd;
#pragma unroll
            for (int k = 0; k < XB; k++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int row = 32 * k + 8 * q + 4 * h;
                    if (row < p.xd && col < p.zd) {
                        if constexpr (ST) {
                            const v4f s = *(const v4f*)(s0 + (size_t)col * p.xd + row);
#pragma unroll
                            for (int w = 0; w < 4; w++) S[k][4 * q + w] = s[w];
                        } else {
#pragma unroll
                            for (int w = 0; w < 4; w++) S[k][4 * q + w] = s0[(size_t)(row + w) * p.zd + col];
                        }
                    }
                }
        }
        // powers: between tokens of the 32 (masked), of a token's entry into the state
        float near[16], enter[16];
#pragma unroll
        for (int v = 0; v < 16; v++) {
            const int row = mix_row(v, h), far = p.back ? row - r : r - row;
            near[v] = far < 0 ? 0.0f : decay_pow(g2, far) * p.near_scale;
            enter[v] = decay_pow(g2, p.back ? row + 1 : 31 - row) * p.add_scale;
        }

        mix_wait();
        __syncthreads();
        const float less = decay_less(g, 32);
        for (int c = 0; c < chunks; c++) {
            const int t0 = start(c), count = min(32, to - t0), buf = c & 1;
            const bool more = c + 1 < chunks;

            // ---- this wavefront's part of the scores: groups of 8 of the head dimension ----
            {
                const unsigned at = r * (XW * 4) + 16 * (h ^ kin_swizzle<XW>(r));
                typedef const __attribute__((address_space(3))) v4f* lds_v4f;
                v16f s = (v16f)(0.0f);
#pragma unroll
                for (int i = 0; i < SHARE; i++) {
                    const int g = wave * SHARE + i;
                    if (NG % ZB == 0 || g < NG) {
                        const unsigned place = (at ^ (32 * (g & 7))) + 256 * (g >> 3);
                        const v4f a = *(lds_v4f)(size_t)(mix_lds(Ys[buf]) + place), b = *(lds_v4f)(size_t)(mix_lds(Xs) + place);
                        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, b.x, s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, b.y, s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, b.z, s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, b.w, s, 0, 0, 0);
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; q++) *(v4f*)&Ps[wave][q * 256 + 4 * lane] = (v4f){s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
            }
            // ---- x . S ----
            v16f o[1] = {(v16f)(0.0f)};
            if (any) {
                const unsigned at = mix_lds(Xs) + r * (XW * 4) + 16 * (h ^ kin_swizzle<XW>(r));
                typedef const __attribute__((address_space(3))) v4f* lds_v4f;
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const v4f b = *(lds_v4f)(size_t)((at ^ (32 * (g & 7))) + 256 * (g >> 3));
#pragma unroll
                    for (int w = 0; w < 4; w++) o[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(S[g / 4][4 * (g % 4) + w], b[w], o[0], 0, 0, 0);
                }
                mix_order<2, NG, 4>();
                o[0] *= decay_pow(g2, p.back ? max(count - 1 - r, 0) : r + 1) * p.far_scale;
            }
            mix_wait();                                             // z
            __syncthreads();
            if (more) fetch_xy(start(c + 1), buf ^ 1);
            __builtin_amdgcn_sched_barrier(0);
            // ---- the near tokens ----
            v16f s;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                v4f sum = *(const v4f*)&Ps[0][q * 256 + 4 * lane];
#pragma unroll
                for (int w = 1; w < ZB; w++) sum += *(const v4f*)&Ps[w][q * 256 + 4 * lane];
#pragma unroll
                for (int w = 0; w < 4; w++) s[4 * q + w] = sum[w] * near[4 * q + w];
            }
            float z[16];
#pragma unroll
            for (int v = 0; v < 16; v++) z[v] = Zs[mix_row(v, h) * ZW + col];
#pragma unroll
            for (int v = 0; v < 16; v++) o[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(z[v], s[v], o[0], 0, 0, 0);
            // ---- into the state ----
            if (more || p.last != nullptr) {
                v16f zw;
                if (count == 32 || p.back) {
#pragma unroll
                    for (int v = 0; v < 16; v++) zw[v] = z[v] * enter[v];
                } else {                                            // the sequence's last, shorter run
#pragma unroll
                    for (int v = 0; v < 16; v++) zw[v] = z[v] * (decay_pow(g2, max(count - 1 - mix_row(v, h), 0)) * p.add_scale);
                }
                if (any) {
                    if constexpr (SLOW) {
                        const float f = count == 32 ? less : decay_less(g, count);
#pragma unroll
                        for (int k = 0; k < XB; k++)
#pragma unroll
                            for (int v = 0; v < 16; v++) S[k][v] = __builtin_fmaf(S[k][v], f, S[k][v]);
                    } else {
                        const float f = decay_pow(g2, count);
#pragma unroll
                        for (int k = 0; k < XB; k++) S[k] *= f;
                    }
                }
                mix_columns_product<XW, XB, true>(S, Ys[buf], zw, cols);
                any = true;
            }
            mix_wait();                                             // the next x and y
            __syncthreads();
            if (more) fetch_z(start(c + 1));
            if (t0 + r < end) mix_store_row<1>(ob + (size_t)(t0 + r) * p.lz.l, o, 1.0f, mine, h);
        }
        // ---- rows behind the sequence's end; the state at the other end ----
        for (int t0 = from + 32 * chunks; t0 < end; t0 += 32)
            if (t0 + r < end)
                for (int d = 4 * h; d < min(mine, 32); d += 8) *(v4f*)(ob + (size_t)(t0 + r) * p.lz.l + d) = (v4f)(0.0f);
        if (p.last != nullptr) {
            float* s1 = p.last + (size_t)nh * p.xd * p.zd;
#pragma unroll
            for (int k = 0; k < XB; k++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int row = 32 * k + mix_row(v, h);
                    if (row < p.xd && col < p.zd) s1[(size_t)row * p.zd + col] = S[k][v];
                }
        }
    };
    if (mix_uniform(decay_slow(g, 32))) along(std::true_type{});
    else along(std::false_type{});
}

// ---------------------------------------------------------------- a segment's own sum
// U[a, b] = sum_t e^{g n(t)} A[t, a] B[t, b], n(t) = tokens behind t in the segment, or (back) t's place in it counted from 1
struct DecayStates {
    const float* A; const float* B;
    MixLayout la, lb;
    const float* g; const int* lens;
    int head, L, ad, bd, segment, segments, back;
    float scale;
    float* U;                 // [image, head, segment][ad][bd]
    int nh;
};

template <int DB, int DC>
__global__ __launch_bounds__(NTHREADS, 2) void decay_states(const DecayStates p) {
    constexpr int DW = DB * 32;
    // the wavefronts share the result: 2 x 2 of them, each TB x TB blocks of 32 x 32 (one block: the first alone)
    constexpr int TB = DC > 2 ? 2 : 1;
    __shared__ __attribute__((aligned(1024))) float As[2][32 * DW];
    __shared__ __attribute__((aligned(1024))) float Bs[2][32 * DW];
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const int lid = xcd_contiguous_id(blockIdx.x, gridDim.x);
    const int segment = mix_uniform(lid / p.nh), nh = lid - segment * p.nh;
    const int n = mix_uniform(nh / p.head), hd = nh - n * p.head;
    const int c0 = segment * p.segment, cnt = min(p.segment, mix_uniform(decay_len(p.lens, n, p.L)) - c0);
    if (cnt <= 0) return;                                // decay_scan does not read it
    const float g2 = decay_log2(p.g[hd]);
    const float* ab = p.A + n * p.la.n + hd * p.la.h + (size_t)c0 * p.la.l;
    const float* bb = p.B + n * p.lb.n + hd * p.lb.h + (size_t)c0 * p.lb.l;
    MixTile<DW, 32, false> at, bt;
    at.init(t, p.la.l, p.ad);
    bt.init(t, p.lb.l, p.bd);
    const unsigned alds = mix_lds(As[0]) + wave * 1024, blds = mix_lds(Bs[0]) + wave * 1024;
    auto fetch = [&](int j0, int into) {
        at.fetch(ab + (size_t)j0 * p.la.l, cnt - j0, p.la.l, alds + into * (32 * DW * 4));
        bt.fetch(bb + (size_t)j0 * p.lb.l, cnt - j0, p.lb.l, blds + into * (32 * DW * 4));
    };
    const int wa = DC > 1 ? (wave >> 1) * TB : 0, wb = DC > 1 ? (wave & 1) * TB : 0;
    const bool works = DC > 1 ? (wa * 32 < p.ad && wb * 32 < p.bd) : wave == 0;
    v16f u[TB][TB];
#pragma unroll
    for (int a = 0; a < TB; a++)
#pragma unroll
        for (int b = 0; b < TB; b++) u[a][b] = (v16f)(0.0f);
    // a token's power: of its place among 32, times that of the 32 in the segment -- both exponents >= 0
    float near[16];
#pragma unroll
    for (int v = 0; v < 16; v++) near[v] = decay_pow(g2, p.back ? mix_row(v, h) + 1 : 31 - mix_row(v, h)) * p.scale;
    fetch(0, 0);
    mix_wait();
    __syncthreads();
    auto step = [&](auto bufc, int j0) {
        constexpr int buf = decltype(bufc)::value;
        if (j0 + 32 < cnt) fetch(j0 + 32, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        if (works) {
            float power[16];
            if (p.back || j0 + 32 <= cnt) {
                const float f = decay_pow(g2, p.back ? j0 : cnt - 32 - j0);
#pragma unroll
                for (int v = 0; v < 16; v++) power[v] = near[v] * f;
            } else {
#pragma unroll
                for (int v = 0; v < 16; v++) power[v] = decay_pow(g2, max(cnt - 1 - j0 - mix_row(v, h), 0)) * p.scale;
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const int row = mix_row(v, h);
                float fa[TB], fb[TB];
#pragma unroll
                for (int a = 0; a < TB; a++) fa[a] = As[buf][row * DW + (wa + a) * 32 + r];
#pragma unroll
                for (int b = 0; b < TB; b++) fb[b] = Bs[buf][row * DW + (wb + b) * 32 + r] * power[v];
#pragma unroll
                for (int a = 0; a < TB; a++)
#pragma unroll
                    for (int b = 0; b < TB; b++) u[a][b] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[a], fb[b], u[a][b], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        mix_wait();
        __syncthreads();
    };
    for (int j0 = 0; j0 < cnt; j0 += 64) {
        step(std::integral_constant<int, 0>{}, j0);
        if (j0 + 32 < cnt) step(std::integral_constant<int, 1>{}, j0 + 32);
    }
    if (!works) return;
    float* U = p.U + ((size_t)nh * p.segments + segment) * p.ad * p.bd;
#pragma unroll
    for (int a = 0; a < TB; a++)
#pragma unroll
        for (int b = 0; b < TB; b++) {
            const int col = (wb + b) * 32 + r;
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const int row = (wa + a) * 32 + mix_row(v, h);
                if (row < p.ad && col < p.bd) U[(size_t)row * p.bd + col] = u[a][b][v];
            }
        }
}

// ---------------------------------------------------------------- over the segments
// In place: U[segment] becomes the state before the segment (back: behind it); the one after the last goes to `last`.
struct DecayScan {
    float* U; const float* first; float* last;
    const float* g; const int* lens;
    int head, L, segment, segments, back, size4;     // size4: float4s of a state
    long long nh;
};
__global__ __launch_bounds__(NTHREADS) void decay_scan(const DecayScan p) {
    const long long x = (long long)blockIdx.x * NTHREADS + threadIdx.x;
    const long long nh = x / p.size4;
    if (nh >= p.nh) return;
    const int e = (int)(x - nh * p.size4);
    const int n = (int)(nh / p.head), hd = (int)(nh - (long long)n * p.head);
    const int len = decay_len(p.lens, n, p.L), used = (len + p.segment - 1) / p.segment;
    const DecayFactor whole = decay_factor(p.g[hd], p.segment), tail = decay_factor(p.g[hd], len - (used - 1) * p.segment);
    v4f* U = (v4f*)p.U + (size_t)nh * p.segments * p.size4 + e;
    v4f s = p.first ? ((const v4f*)p.first)[nh * p.size4 + e] : (v4f)(0.0f);
    constexpr int AHEAD = 8;       // loads in flight: each would otherwise wait for the one before
    for (int k0 = 0; k0 < used; k0 += AHEAD) {
        v4f u[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int k = min(k0 + i, used - 1);
            u[i] = U[(size_t)(p.back ? used - 1 - k : k) * p.size4];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (k0 + i >= used) break;
            const int c = p.back ? used - 1 - (k0 + i) : k0 + i;
            U[(size_t)c * p.size4] = s;
            const DecayFactor f = c == used - 1 ? tail : whole;
            s = s * f.f + (s * f.keep + u[i]);
        }
    }
    if (p.last) ((v4f*)p.last)[nh * p.size4 + e] = s;
}

// ---------------------------------------------------------------- few tokens
struct DecaySteps {
    const float* Q; const float* K; const float* V; float* Y;
    MixLayout q, k, v, y;
    const float* g; const int* lens;
    const float* first; float* last;
    int head, L, dk, dv, slabs;
    float scale;
};
// A thread holds 4 columns of rows row0, row0 + LANES, ... of the state; a token's output is added over the row groups of a
// wavefront by exchange and over the wavefronts through LDS.  COLS: columns of the state per workgroup -- 32, and 64 (256
// contiguous bytes a row) for states that pass the caches by: 256 x 32 states of 128 x 128 in 193 us instead of 205, but
// smaller batches are level or behind with it.
template <bool NT, int COLS>
__global__ __launch_bounds__(NTHREADS) void decay_steps(const DecaySteps p) {
    constexpr int ACROSS = COLS / 4, LANES = NTHREADS / ACROSS, STEP_ROWS = 128 / LANES;
    __shared__ __attribute__((aligned(16))) float part[2][4][COLS];
    const int t = threadIdx.x, wave = t >> 6;
    const int nh = blockIdx.x / p.slabs, slab = blockIdx.x - nh * p.slabs;
    const int n = nh / p.head, hd = nh - n * p.head;
    const float g = p.g[hd];
    const int len = decay_len(p.lens, n, p.L);
    const int col = slab * COLS + 4 * (t % ACROSS), row0 = t / ACROSS;
    const bool mine = col < p.dv;
    const size_t base = (size_t)nh * p.dk * p.dv + col;
    v4f s[STEP_ROWS];
#pragma unroll
    for (int a = 0; a < STEP_ROWS; a++) {
        const int row = row0 + LANES * a;
        s[a] = (mine && row < p.dk && p.first) ? stream_load4<NT>(p.first + base + (size_t)row * p.dv) : (v4f)(0.0f);
    }
    const float* q = p.Q + n * p.q.n + hd * p.q.h;
    const float* k = p.K + n * p.k.n + hd * p.k.h;
    const float* v = p.V + n * p.v.n + hd * p.v.h;
    float* y = p.Y + n * p.y.n + hd * p.y.h;
    // a token's operands are read while the one before is worked on
    v4f vn = (v4f)(0.0f);
    float kn[STEP_ROWS] = {}, qn[STEP_ROWS] = {};
    auto read = [&](int i) {
        if (mine) vn = *(const v4f*)(v + (size_t)i * p.v.l + col);
#pragma unroll
        for (int a = 0; a < STEP_ROWS; a++) {
            const int row = row0 + LANES * a;
            if (row < p.dk) {
                kn[a] = k[(size_t)i * p.k.l + row];
                qn[a] = q[(size_t)i * p.q.l + row];
            }
        }
    };
    if (len > 0) read(0);
    const DecayFactor lam = decay_factor(g, 1);
    for (int i = 0; i < len; i++) {
        const v4f vv = vn;
        v4f out = (v4f)(0.0f);
        float qi[STEP_ROWS];
#pragma unroll
        for (int a = 0; a < STEP_ROWS; a++) {
            qi[a] = qn[a];
            s[a] = vv * kn[a] + (s[a] * lam.f + s[a] * lam.keep);
        }
        if (i + 1 < len) read(i + 1);
#pragma unroll
        for (int a = 0; a < STEP_ROWS; a++) out += s[a] * qi[a];
#pragma unroll
        for (int x = ACROSS; x < 64; x <<= 1)
#pragma unroll
            for (int u = 0; u < 4; u++) out[u] += __shfl_xor(out[u], x, 64);
        if ((t & 63) < ACROSS) *(v4f*)&part[i & 1][wave][4 * (t % ACROSS)] = out;
        __syncthreads();                      // one a token: the next token writes the other half
        if (t < ACROSS && mine) {
            const v4f sum = (*(const v4f*)&part[i & 1][0][4 * t] + *(const v4f*)&part[i & 1][1][4 * t]) +
                            (*(const v4f*)&part[i & 1][2][4 * t] + *(const v4f*)&part[i & 1][3][4 * t]);
            *(v4f*)(y + (size_t)i * p.y.l + col) = sum * p.scale;
        }
    }
    if (t < ACROSS && mine)
        for (int i = len; i < p.L; i++) *(v4f*)(y + (size_t)i * p.y.l + col) = (v4f)(0.0f);
    if (p.last && mine) {
#pragma unroll
        for (int a = 0; a < STEP_ROWS; a++) {
            const int row = row0 + LANES * a;
            if (row < p.dk) stream_store4<NT>(p.last + base + (size_t)row * p.dv, s[a]);
        }
    }
}

// ---------------------------------------------------------------- host side
// Up to here the recurrence: 8 tokens of 32 heads of 128 in 9.3 us and of 64 x 32 in 84 (the walk: 14.1 and 98), 12 in 12.0 and
// 108 (14.1 and 104), 16 in 14.8 and 133 (14.1 and 108).
constexpr int STEPS_MAX = 12;

// The workgroups of decay_walk that the chip holds, x being xd columns wide and z zd: two a compute unit where either is above 64
// (LDS).  500 pairs of 128 x 64 and 4096 tokens take 885 us whole; cut in two, as if four a unit had room, 1871.  (At 64 x 32 LDS
// holds five, not eight, but with five the estimate below is no better: 170 us for 475 at 960 pairs, 268 for 205 at 1440.)
constexpr int decay_slots(int xd, int zd) { return xd > 64 || zd > 64 ? 512 : zd > 32 ? 1024 : 2048; }
// How a sequence is cut: into as many segments as fill the chip with workgroups, where that is taken to be faster than walking along
// it whole -- the segments' sums cost one product more to the walk's two and a half, and two launches (3.7 and 12 runs of 32
// tokens' time).  Cut against whole: 16 heads of 128 and 300 tokens 30 us against 66, 4 x 16 of 64 and 1000 43 against 122,
// 8 x 16 of 128 and 2000 289 against 408.  The estimate counts rounds of workgroups and does not know that
// one alone on a compute unit walks faster than two: from half a round on it cuts too early (16 x 16 of 128 and 2000 tokens: 557
// against 416).
// At most 64 segments, which bounds the work buffer: one head of 128 and 32768 tokens takes 152 us (32: 280; 256 would take
// 82), 4 heads 160 (284; 158), 16 heads 540 (547; 546).
struct DecayCut { int segment, segments; };
DecayCut decay_cut(int N, int head, int L, int slots) {
    const long long nh = (long long)N * head, chunks = (L + 31LL) / 32;
    DecayCut best = {(int)(chunks * 32), 1};
    double least = 0.0;
    for (long long want = 1; want <= 64; want++) {
        const long long per = (chunks + want - 1) / want, segments = (chunks + per - 1) / per;
        if (segments != want) continue;
        const double walk = (double)((nh * segments + slots - 1) / slots) * per;
        const double cost = segments == 1 ? 2.5 * walk : 3.7 * walk + 12.0;
        if (want == 1 || cost < least) {
            least = cost;
            best.segment = (int)(per * 32);
            best.segments = (int)segments;
        }
    }
    return best;
}

long long decay_state_bytes(int N, int head, const DecayCut& cut, int dK4, int dV4) {
    return cut.segments == 1 ? 0 : (long long)N * head * cut.segments * dK4 * dV4 * 4;
}

bool decay_arguments_ok(int N, int head, int L, int dK4, int dV4) {
    if (N <= 0 || head <= 0 || L <= 0 || dK4 <= 0 || dV4 <= 0 || (dK4 & 3) || (dV4 & 3) || dK4 > 128 || dV4 > 128) return false;
    const long long row = (long long)head * (dK4 > dV4 ? dK4 : dV4);
    // a tile's offsets are 32-bit bytes, positions 32-bit, image-head pairs 25 bits
    return L < 0x3fffff00 && row * 32 * 4 < 0x7ffffff0LL && (long long)N * head * 64 < 0x7fffffffLL &&
           (long long)N * head * dK4 * dV4 / 4 < 0x7fffffffLL * 128;
}
// a walk has a wavefront for 32 columns of z, of a workgroup for each pair and segment (which are many only where the pairs are
// few); decay_steps a workgroup of four for 64 columns of V where it has to
bool decay_walk_fits(int N, int head, int zd) { return mix_launch_fits((long long)N * head, 64 * ((zd + 31) / 32)); }
bool decay_steps_fit(int N, int head, int dV4, int cols) {
    return mix_launch_fits((long long)N * head * ((dV4 + cols - 1) / cols), NTHREADS);
}
bool decay_forward_ok(int N, int head, int L, int dK4, int dV4) {
    return decay_arguments_ok(N, head, L, dK4, dV4) && (L <= STEPS_MAX ? decay_steps_fit(N, head, dV4, 64) : decay_walk_fits(N, head, dV4));
}
bool decay_backward_ok(int N, int head, int L, int dK4, int dV4) {
    return decay_arguments_ok(N, head, L, dK4, dV4) && decay_walk_fits(N, head, dK4 > dV4 ? dK4 : dV4);
}

hipError_t launch_states(hipStream_t s, const float* A, MixLayout la, int ad, const float* B, MixLayout lb, int bd, const float* g,
                         const int* lens, int N, int head, int L, const DecayCut& cut, int back, float scale, float* U) {
    DecayStates p = {A, B, la, lb, g, lens, head, L, ad, bd, cut.segment, cut.segments, back, scale, U, N * head};
    const dim3 grid((unsigned)((long long)N * head * cut.segments)), block(NTHREADS);
    switch (((ad > bd ? ad : bd) + 31) / 32) {
        case 1: hipLaunchKernelGGL((decay_states<1, 1>), grid, block, 0, s, p); break;
        case 2: hipLaunchKernelGGL((decay_states<2, 2>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((decay_states<4, 4>), grid, block, 0, s, p); break;
    }
    return hipGetLastError();
}

hipError_t launch_scan(hipStream_t s, float* U, const float* first, float* last, const float* g, const int* lens, int N, int head,
                       int L, const DecayCut& cut, int back, int size) {
    DecayScan p = {U, first, last, g, lens, head, L, cut.segment, cut.segments, back, size / 4, (long long)N * head};
    const long long items = p.nh * p.size4;
    hipLaunchKernelGGL(decay_scan, dim3((unsigned)((items + NTHREADS - 1) / NTHREADS)), dim3(NTHREADS), 0, s, p);
    return hipGetLastError();
}

template <bool ST>
hipError_t launch_walk(hipStream_t s, const DecayWalk& p) {
    const dim3 grid((unsigned)((long long)p.nh * p.segments));
    const int xb = (p.xd + 31) / 32, zb = (p.zd + 31) / 32;
#define WALK(XB, ZB) hipLaunchKernelGGL((decay_walk<XB, ZB, ST>), grid, dim3(64 * ZB), 0, s, p)
#define WALK_Z(XB)                                                                                     \
    do {                                                                                               \
        if (zb == 1) WALK(XB, 1); else if (zb == 2) WALK(XB, 2); else if (zb == 3) WALK(XB, 3); else WALK(XB, 4); \
    } while (0)
    if (xb == 1) WALK_Z(1);
    else if (xb == 2) WALK_Z(2);
    else WALK_Z(4);
#undef WALK_Z
#undef WALK
    return hipGetLastError();
}

}  // namespace
}  // namespace dragon

using namespace dragon;

extern "C" {

int64_t dragon_Cuda_linear_attention_bufsize(int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4) {
    if (!decay_forward_ok(N, head, L, dK4, dV4)) return -1;
    return L <= STEPS_MAX ? 0 : decay_state_bytes(N, head, decay_cut(N, head, L, decay_slots(dK4, dV4)), dK4, dV4);
}
int64_t dragon_Cuda_linear_attention_backward_bufsize(int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4) {
    if (!decay_backward_ok(N, head, L, dK4, dV4)) return -1;
    return 2 * decay_state_bytes(N, head, decay_cut(N, head, L, decay_slots(dK4, dK4 > dV4 ? dK4 : dV4)), dK4, dV4);
}

int dragon_Cuda_linear_attention_forward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV, int64_t dDecay,
                                         int64_t dState, int64_t dY, int64_t dStateOut, int64_t dLens, int64_t dBuf,
                                         int64_t buf_size, int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4,
                                         int32_t head_inner, float scale) {
    if (streams == nullptr || length < 1 || length > 10) return hipErrorInvalidValue;
    if (dQ == 0 || dK == 0 || dV == 0 || dDecay == 0 || dY == 0 || !mix_aligned16(dQ) || !mix_aligned16(dK) || !mix_aligned16(dV) ||
        !mix_aligned16(dY) || !mix_aligned16(dState) || !mix_aligned16(dStateOut) || (dDecay & 3) || (dLens & 3))
        return hipErrorInvalidValue;
    if (!decay_forward_ok(N, head, L, dK4, dV4) || !(scale - scale == 0.0f)) return hipErrorInvalidValue;
    const long long need = dragon_Cuda_linear_attention_bufsize(N, head, L, dK4, dV4);
    if (need > 0 && (dBuf == 0 || !mix_aligned16(dBuf) || buf_size < need)) return hipErrorInvalidValue;
    const float* Q = (const float*)(intptr_t)dQ; const float* K = (const float*)(intptr_t)dK; const float* V = (const float*)(intptr_t)dV;
    const float* first = (const float*)(intptr_t)dState; const float* g = (const float*)(intptr_t)dDecay;
    float* Y = (float*)(intptr_t)dY; float* last = (float*)(intptr_t)dStateOut; float* U = (float*)(intptr_t)dBuf;
    const int* lens = (const int*)(intptr_t)dLens;
    const MixLayout lk = mix_layout(head_inner, head, L, dK4), lv = mix_layout(head_inner, head, L, dV4);
    const size_t state = (size_t)dK4 * dV4;
    split_ledger_touch(Y, (size_t)N * head * L * dV4 * 4);
    if (last != nullptr) split_ledger_touch(last, (size_t)N * head * state * 4);
    if (need > 0) split_ledger_touch(U, (size_t)need);
    hipStream_t s = (hipStream_t)(intptr_t)streams[0];
    if (L <= STEPS_MAX) {
        // (also where the states are so many that only workgroups of 64 columns fit a launch)
        const bool nt = (first != nullptr && last != nullptr && stream_nt(first, last, (long long)N * head * state * 4)) ||
                        !decay_steps_fit(N, head, dV4, 32);
        const int cols = nt ? 64 : 32;
        DecaySteps p = {Q, K, V, Y, lk, lk, lv, lv, g, lens, first, last, head, L, dK4, dV4, (dV4 + cols - 1) / cols, scale};
        const dim3 grid((unsigned)((long long)N * head * p.slabs));
        if (nt) hipLaunchKernelGGL((decay_steps<true, 64>), grid, dim3(NTHREADS), 0, s, p);
        else hipLaunchKernelGGL((decay_steps<false, 32>), grid, dim3(NTHREADS), 0, s, p);
        return hipGetLastError();
    }
    const DecayCut cut = decay_cut(N, head, L, decay_slots(dK4, dV4));
    DecayWalk p = {Q, K, V, Y, lk, lv, g, lens, head, L, dK4, dV4, cut.segment, cut.segments, 0, scale, scale, 1.0f,
                   first, last, N * head};
    if (cut.segments > 1) {
        hipError_t e = launch_states(s, K, lk, dK4, V, lv, dV4, g, lens, N, head, L, cut, 0, 1.0f, U);
        if (e == hipSuccess) e = launch_scan(s, U, first, last, g, lens, N, head, L, cut, 0, (int)state);
        if (e != hipSuccess) return e;
        p.state = U;
        p.last = nullptr;
    }
    return launch_walk<false>(s, p);
}

int dragon_Cuda_linear_attention_backward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV, int64_t dDecay,
                                          int64_t dState, int64_t dDeltaY, int64_t dDeltaStateOut, int64_t dDeltaQ, int64_t dDeltaK,
                                          int64_t dDeltaV, int64_t dDeltaState, int64_t dLens, int64_t dBuf, int64_t buf_size,
                                          int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4, int32_t head_inner,
                                          float scale) {
    if (streams == nullptr || length < 1 || length > 10) return hipErrorInvalidValue;
    if (dQ == 0 || dK == 0 || dV == 0 || dDecay == 0 || dDeltaY == 0 || dDeltaQ == 0 || dDeltaK == 0 || dDeltaV == 0 ||
        !mix_aligned16(dQ) || !mix_aligned16(dK) || !mix_aligned16(dV) || !mix_aligned16(dState) || !mix_aligned16(dDeltaY) ||
        !mix_aligned16(dDeltaStateOut) || !mix_aligned16(dDeltaQ) || !mix_aligned16(dDeltaK) || !mix_aligned16(dDeltaV) ||
        !mix_aligned16(dDeltaState) || (dDecay & 3) || (dLens & 3))
        return hipErrorInvalidValue;
    if (!decay_backward_ok(N, head, L, dK4, dV4) || !(scale - scale == 0.0f)) return hipErrorInvalidValue;
    const DecayCut cut = decay_cut(N, head, L, decay_slots(dK4, dK4 > dV4 ? dK4 : dV4));   // (either width is x in one of the walks)
    const long long need = 2 * decay_state_bytes(N, head, cut, dK4, dV4);
    if (need > 0 && (dBuf == 0 || !mix_aligned16(dBuf) || buf_size < need)) return hipErrorInvalidValue;
    const float* Q = (const float*)(intptr_t)dQ; const float* K = (const float*)(intptr_t)dK; const float* V = (const float*)(intptr_t)dV;
    const float* G = (const float*)(intptr_t)dDeltaY; const float* g = (const float*)(intptr_t)dDecay;
    const float* first = (const float*)(intptr_t)dState; const float* dlast = (const float*)(intptr_t)dDeltaStateOut;
    float* gQ = (float*)(intptr_t)dDeltaQ; float* gK = (float*)(intptr_t)dDeltaK; float* gV = (float*)(intptr_t)dDeltaV;
    float* gfirst = (float*)(intptr_t)dDeltaState;
    const int* lens = (const int*)(intptr_t)dLens;
    const long long state = (long long)dK4 * dV4;
    float* S = need > 0 ? (float*)(intptr_t)dBuf : nullptr;
    float* R = need > 0 ? S + (size_t)N * head * cut.segments * state : nullptr;
    const MixLayout lk = mix_layout(head_inner, head, L, dK4), lv = mix_layout(head_inner, head, L, dV4);
    split_ledger_touch(gQ, (size_t)N * head * L * dK4 * 4);
    split_ledger_touch(gK, (size_t)N * head * L * dK4 * 4);
    split_ledger_touch(gV, (size_t)N * head * L * dV4 * 4);
    if (gfirst != nullptr) split_ledger_touch(gfirst, (size_t)N * head * state * 4);
    if (need > 0) split_ledger_touch(S, (size_t)need);
    hipStream_t s = (hipStream_t)(intptr_t)streams[0];
    const float* before = first;       // what the segments begin with, and end with
    const float* behind = dlast;
    hipError_t e = hipSuccess;
    if (cut.segments > 1) {
        e = launch_states(s, K, lk, dK4, V, lv, dV4, g, lens, N, head, L, cut, 0, 1.0f, S);
        if (e == hipSuccess) e = launch_scan(s, S, first, nullptr, g, lens, N, head, L, cut, 0, (int)state);
        if (e == hipSuccess) e = launch_states(s, Q, lk, dK4, G, lv, dV4, g, lens, N, head, L, cut, 1, scale, R);
        if (e == hipSuccess) e = launch_scan(s, R, dlast, gfirst, g, lens, N, head, L, cut, 1, (int)state);
        if (e != hipSuccess) return e;
        before = S;
        behind = R;
    }
    DecayWalk p = {G, V, K, gQ, lv, lk, g, lens, head, L, dV4, dK4, cut.segment, cut.segments, 0, scale, scale, 1.0f,
                   before, nullptr, N * head};
    e = launch_walk<true>(s, p);
    p.back = 1; p.far_scale = 1.0f; p.add_scale = scale;
    p.state = behind;
    p.x = V; p.y = G; p.z = Q; p.out = gK;
    if (e == hipSuccess) e = launch_walk<true>(s, p);
    p.x = K; p.y = Q; p.z = G; p.out = gV; p.lx = lk; p.lz = lv; p.xd = dK4; p.zd = dV4;
    p.last = cut.segments == 1 ? gfirst : nullptr;
    if (e == hipSuccess) e = launch_walk<false>(s, p);
    return e;
}

}  // extern "C"
