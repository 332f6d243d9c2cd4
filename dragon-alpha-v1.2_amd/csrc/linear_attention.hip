// Linear attention with a decay for each head: a state S[dk, dv] per (image, head) that forgets by a constant factor a token,
//     S_t = e^g S_{t-1} + K[t]^T V[t],     Y[t] = scale * Q[t] S_t            (g <= 0, one per head)
// and its gradient.
//
// Few tokens (decay_steps): the recurrence itself, the state in registers; bound by reading and writing the states.
// Many tokens: chunks of C.  With S_c the state before chunk c and t the token's place in it,
//     Y[t] = scale * (e^{g(t+1)} Q[t] S_c  +  sum_{j <= t} e^{g(t-j)} <Q[t], K[j]> V[j])
// in three launches: decay_states adds up each chunk's own K^T V, decay_scan runs over the chunks and leaves S_c in their
// place, decay_mix multiplies.  The chunks are independent in the first and the last, so a single long sequence fills the
// chip; bound by the FP32 matrix pipe, then by memory (a longer chunk: more products inside it, fewer states to move).
//
// The gradient is the same three launches with other operands (G = gradient of Y, sums over j >= t in the last two):
//     dQ[t] = scale sum e^{g(t-j)} <G[t], V[j]> K[j] + ...  S_c^T           the states of the forward pass again
//     dK[t] = scale sum e^{g(j-t)} <V[t], G[j]> Q[j] + ...  R_c^T           R: the same sum from the sequence's end,
//     dV[t] = scale sum e^{g(j-t)} <K[t], Q[j]> G[j] + ...  R_c             over Q^T G, starting with the gradient of the last state
// so decay_mix takes its operands x, y, z by name, a direction, and the state either way round.
//
// Every power e^{g n} is computed as such (n >= 0: it cannot overflow), never as a quotient of two powers.  States, sums and
// powers are FP32; the exponent g n is rounded once, which is an error of |g n| 2^-24 in a factor e^{g n}.
#include "token_mixer.h"
#include "runtime_internal.h"
#include "../../include/dragon_hip_gemm.h"

namespace dragon {
namespace {

constexpr int TQ = 128;       // tokens per workgroup of decay_mix: 32 per wavefront
constexpr int MAX_CHUNK = 256;

struct DecayParams {
    const float* x; const float* y; const float* z; float* out;   // [L, xd], [L, xd], [L, zd], [L, zd] per (image, head)
    MixLayout lx, ly, lz, lo;
    const float* g; const int* lens;
    int head, L, xd, zd, C, chunks;
    int back;                  // sums over j >= t instead of j <= t
    float near_scale, far_scale;   // factors on the sum inside the chunk and on the state's share
    const float* state;        // the state before each chunk, [image, head, chunk]; null: none at all
    int empty_first;           // the state at the sequence's beginning (back: at its end) is zero
    long long state_nh, state_c;   // its strides
    int tiles, nh;
};

__device__ __forceinline__ float decay_log2(const float* g, int hd) {
    // not below -1e30: 0 * g has to be 0 where the head forgets at once (g = -infinity)
    return fmaxf(g[hd] * MIX_LOG2E, -1.0e30f);
}
__device__ __forceinline__ float decay_pow(float g2, int n) { return __builtin_amdgcn_exp2f(g2 * (float)n); }
__device__ __forceinline__ int decay_len(const int* lens, int n, int L) { return lens ? min(max(lens[n], 0), L) : L; }

// ---------------------------------------------------------------- inside the chunks, and the state's share
// ST: the state lies [zd][xd] (its transpose is what multiplies x)
template <int DB, int DC, bool ST>
__global__ __launch_bounds__(NTHREADS, 2) void decay_mix(const DecayParams p) {
    constexpr int DW = DB * 32, NG = DC * 4;
    __shared__ __attribute__((aligned(16))) float Ys[2][32 * DW];
    __shared__ __attribute__((aligned(16))) float Zs[2][32 * DW];
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const int lid = xcd_contiguous_id(blockIdx.x, gridDim.x);
    const int tile = mix_uniform(lid / p.nh), nh = lid - tile * p.nh;
    const int n = mix_uniform(nh / p.head), hd = nh - n * p.head;
    const int len = mix_uniform(decay_len(p.lens, n, p.L));
    // Inside a chunk the later (back: the earlier) 32 tokens have the most to do.  The workgroups that share a compute unit
    // give them to different wavefronts, so that no SIMD has all the work.
    const int q0 = tile * TQ, w0 = q0 + 32 * ((blockIdx.x >> 8) & 1 ? 3 - wave : wave), i = w0 + r;
    const int chunk = mix_uniform(q0 / p.C), c0 = chunk * p.C, c1 = min(c0 + p.C, len);
    const float g2 = decay_log2(p.g, hd);
    const float* xb = p.x + n * p.lx.n + hd * p.lx.h;
    const float* yb = p.y + n * p.ly.n + hd * p.ly.h;
    const float* zb = p.z + n * p.lz.n + hd * p.lz.h;

    v4f xf[NG];
    mix_load_cols<NG>(xf, xb + (size_t)min(i, p.L - 1) * p.lx.l, i < len, p.xd, h);
    v16f o[DC];
#pragma unroll
    for (int b = 0; b < DC; b++) o[b] = (v16f)(0.0f);

    MixColumns<DW, false> zcols;
    zcols.init(r, h);

    const unsigned ylds = mix_lds(Ys[0]) + wave * 1024, zlds = mix_lds(Zs[0]) + wave * 1024;
    constexpr unsigned TILE = 32 * DW * 4;

    // ---- x . S: 32 rows of the state per step ----
    const bool first_chunk = p.back ? c1 == len : chunk == 0;
    if (q0 < len && p.state != nullptr && !(first_chunk && p.empty_first)) {
        const float* sb = p.state + nh * p.state_nh + chunk * p.state_c;
        if constexpr (ST) {
            MixTile<DW, 32, true> st;
            st.init(t, p.xd, p.xd);
            st.fetch(sb, p.zd, p.xd, ylds);
            static_for<DC>([&](auto bc) {
                constexpr int b = decltype(bc)::value;
                mix_wait();
                __syncthreads();
                if (b + 1 < DC) st.fetch(sb + (size_t)(b + 1) * 32 * p.xd, p.zd - (b + 1) * 32, p.xd, ylds + ((b + 1) & 1) * TILE);
                __builtin_amdgcn_sched_barrier(0);
                mix_rows_product<DW, NG>(o[b], Ys[b & 1], xf, r, h);
            });
        } else {
            MixTile<DW, 32, false> st;
            st.init(t, p.zd, p.zd);
            st.fetch(sb, p.xd, p.zd, zlds);
            static_for<DC>([&](auto bc) {
                constexpr int b = decltype(bc)::value;
                mix_wait();
                __syncthreads();
                if (b + 1 < DC) st.fetch(sb + (size_t)(b + 1) * 32 * p.zd, p.xd - (b + 1) * 32, p.zd, zlds + ((b + 1) & 1) * TILE);
                __builtin_amdgcn_sched_barrier(0);
                v16f w;
#pragma unroll
                for (int v = 0; v < 16; v++) w[v] = xf[4 * b + v / 4][v % 4];
                mix_columns_product<DW, DC, false>(o, Zs[b & 1], w, zcols, r, h);
            });
        }
        const float f = decay_pow(g2, max(p.back ? c1 - 1 - i : i - c0 + 1, 0)) * p.far_scale;
#pragma unroll
        for (int b = 0; b < DC; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) o[b][v] *= f;
        __syncthreads();
    }

    // ---- the chunk's own tokens, 32 per step ----
    const int from = p.back ? q0 : c0, to = q0 < len ? (p.back ? c1 : min(q0 + TQ, len)) : from;
    MixTile<DW, 32, true> yt;
    MixTile<DW, 32, false> zt;
    yt.init(t, p.ly.l, p.xd);
    zt.init(t, p.lz.l, p.zd);
    auto fetch = [&](int j0, int into) {
        yt.fetch(yb + (size_t)j0 * p.ly.l, to - j0, p.ly.l, ylds + into * TILE);
        zt.fetch(zb + (size_t)j0 * p.lz.l, to - j0, p.lz.l, zlds + into * TILE);
    };
    // e^(g distance) inside the wavefront's own 32 tokens, and for 32 tokens that lie at least 32 away but for a factor that
    // is the same for all of them: every power here is >= 0
    float own[16], near[16];
#pragma unroll
    for (int v = 0; v < 16; v++) {
        const int far = p.back ? mix_row(v, h) - r : r - mix_row(v, h);
        own[v] = far < 0 ? 0.0f : decay_pow(g2, far) * p.near_scale;
        near[v] = decay_pow(g2, 31 + far) * p.near_scale;
    }
    if (from < to) fetch(from, 0);
    mix_wait();
    __syncthreads();
    auto step = [&](auto bufc, int j0) {
        constexpr int buf = decltype(bufc)::value;
        if (j0 + 32 < to) fetch(j0 + 32, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        const int away = p.back ? j0 - w0 : w0 - j0;        // a multiple of 32
        if (away >= 0) {
            v16f s = (v16f)(0.0f);
            mix_rows_product<DW, NG>(s, Ys[buf], xf, r, h);
            if (away > 0) {
                const float f = decay_pow(g2, away - 31);
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] *= near[v] * f;
            } else {
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] *= own[v];
            }
            mix_columns_product<DW, DC, false>(o, Zs[buf], s, zcols, r, h);
        }
        mix_wait();
        __syncthreads();
    };
    for (int j0 = from; j0 < to; j0 += 64) {
        step(std::integral_constant<int, 0>{}, j0);
        if (j0 + 32 < to) step(std::integral_constant<int, 1>{}, j0 + 32);
    }
    if (i < p.L) mix_store_row<DC>(p.out + n * p.lo.n + hd * p.lo.h + (size_t)i * p.lo.l, o, 1.0f, p.zd, h);
}

// ---------------------------------------------------------------- a chunk's own sum
// U[a, b] = sum_t e^{g n(t)} A[t, a] B[t, b], n(t) = tokens behind t in the chunk, or (back) t's place in it counted from 1
struct DecayStates {
    const float* A; const float* B;
    MixLayout la, lb;
    const float* g; const int* lens;
    int head, L, ad, bd, C, chunks, back;
    float scale;
    float* U;                 // [image, head, chunk][ad][bd]
    int nh;
};

template <int DB, int DC>
__global__ __launch_bounds__(NTHREADS, 2) void decay_states(const DecayStates p) {
    constexpr int DW = DB * 32;
    // the wavefronts share the result: 2 x 2 of them, each TB x TB blocks of 32 x 32 (one block: the first alone)
    constexpr int TB = DC > 2 ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float As[2][32 * DW];
    __shared__ __attribute__((aligned(16))) float Bs[2][32 * DW];
    __shared__ __attribute__((aligned(16))) float Ws[MAX_CHUNK];      // a token's power
    const int t = threadIdx.x, lane = t & 63, wave = mix_uniform(t >> 6), r = lane & 31, h = lane >> 5;
    const int lid = xcd_contiguous_id(blockIdx.x, gridDim.x);
    const int chunk = mix_uniform(lid / p.nh), nh = lid - chunk * p.nh;
    const int n = mix_uniform(nh / p.head), hd = nh - n * p.head;
    const int c0 = chunk * p.C, cnt = min(p.C, mix_uniform(decay_len(p.lens, n, p.L)) - c0);
    if (cnt <= 0) return;                                // decay_scan does not read it
    const float g2 = decay_log2(p.g, hd);
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
    for (int j = t; j < MAX_CHUNK; j += NTHREADS) Ws[j] = decay_pow(g2, max(p.back ? j + 1 : cnt - 1 - j, 0)) * p.scale;
    fetch(0, 0);
    mix_wait();
    __syncthreads();
    int buf = 0;
    for (int j0 = 0; j0 < cnt; j0 += 32) {
        if (j0 + 32 < cnt) fetch(j0 + 32, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        if (works) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const v4f w = *(const v4f*)&Ws[j0 + 8 * q + 4 * h];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int row = mix_row(4 * q + x, h);
                    float fa[TB], fb[TB];
#pragma unroll
                    for (int a = 0; a < TB; a++) fa[a] = As[buf][row * DW + (wa + a) * 32 + r];
#pragma unroll
                    for (int b = 0; b < TB; b++) fb[b] = Bs[buf][row * DW + (wb + b) * 32 + r] * w[x];
#pragma unroll
                    for (int a = 0; a < TB; a++)
#pragma unroll
                        for (int b = 0; b < TB; b++) u[a][b] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[a], fb[b], u[a][b], 0, 0, 0);
                }
            }
        }
        mix_wait();
        __syncthreads();
        buf ^= 1;
    }
    if (!works) return;
    float* U = p.U + ((size_t)nh * p.chunks + chunk) * p.ad * p.bd;
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

// ---------------------------------------------------------------- over the chunks
// In place: U[chunk] becomes the state before the chunk (back: behind it); the one after the last goes to `last`.
struct DecayScan {
    float* U; const float* first; float* last;
    const float* g; const int* lens;
    int head, L, C, chunks, back, size4;     // size4: float4s of a state
    long long nh;
};
__global__ __launch_bounds__(NTHREADS) void decay_scan(const DecayScan p) {
    const long long x = (long long)blockIdx.x * NTHREADS + threadIdx.x;
    const long long nh = x / p.size4;
    if (nh >= p.nh) return;
    const int e = (int)(x - nh * p.size4);
    const int n = (int)(nh / p.head), hd = (int)(nh - (long long)n * p.head);
    const int len = decay_len(p.lens, n, p.L), used = (len + p.C - 1) / p.C;
    const float g2 = decay_log2(p.g, hd);
    const float whole = decay_pow(g2, p.C), tail = decay_pow(g2, len - (used - 1) * p.C);
    v4f* U = (v4f*)p.U + (size_t)nh * p.chunks * p.size4 + e;
    v4f s = p.first ? ((const v4f*)p.first)[nh * p.size4 + e] : (v4f)(0.0f);
    v4f next = (v4f)(0.0f);
    if (used > 0) next = U[(size_t)(p.back ? used - 1 : 0) * p.size4];
    for (int k = 0; k < used; k++) {
        const int c = p.back ? used - 1 - k : k;
        const v4f u = next;
        if (k + 1 < used) next = U[(size_t)(p.back ? c - 1 : c + 1) * p.size4];
        U[(size_t)c * p.size4] = s;
        s = s * (c == used - 1 ? tail : whole) + u;
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
constexpr int STEP_COLS = 32;                 // columns of the state per workgroup
constexpr int STEP_ROWS = 128 / (NTHREADS / (STEP_COLS / 4));   // rows of the state per thread
// A thread holds 4 columns of rows row0, row0 + 32, ... of the state; a token's output is added over the 8 row groups of a
// wavefront by exchange and over the wavefronts through LDS.
__global__ __launch_bounds__(NTHREADS) void decay_steps(const DecaySteps p) {
    __shared__ __attribute__((aligned(16))) float part[2][4][STEP_COLS];
    const int t = threadIdx.x, wave = t >> 6;
    const int nh = blockIdx.x / p.slabs, slab = blockIdx.x - nh * p.slabs;
    const int n = nh / p.head, hd = nh - n * p.head;
    const int len = decay_len(p.lens, n, p.L);
    const int col = slab * STEP_COLS + 4 * (t & 7), row0 = t >> 3;
    const bool mine = col < p.dv;
    const float lam = decay_pow(decay_log2(p.g, hd), 1);
    const size_t base = (size_t)nh * p.dk * p.dv + col;
    v4f s[STEP_ROWS];
#pragma unroll
    for (int a = 0; a < STEP_ROWS; a++) {
        const int row = row0 + 32 * a;
        s[a] = (mine && row < p.dk && p.first) ? *(const v4f*)(p.first + base + (size_t)row * p.dv) : (v4f)(0.0f);
    }
    const float* q = p.Q + n * p.q.n + hd * p.q.h;
    const float* k = p.K + n * p.k.n + hd * p.k.h;
    const float* v = p.V + n * p.v.n + hd * p.v.h;
    float* y = p.Y + n * p.y.n + hd * p.y.h;
    for (int i = 0; i < len; i++) {
        const v4f vv = mine ? *(const v4f*)(v + (size_t)i * p.v.l + col) : (v4f)(0.0f);
        v4f out = (v4f)(0.0f);
#pragma unroll
        for (int a = 0; a < STEP_ROWS; a++) {
            const int row = row0 + 32 * a;
            if (row < p.dk) {
                s[a] = s[a] * lam + vv * k[(size_t)i * p.k.l + row];
                out += s[a] * q[(size_t)i * p.q.l + row];
            }
        }
#pragma unroll
        for (int x = 8; x < 64; x <<= 1)
#pragma unroll
            for (int u = 0; u < 4; u++) out[u] += __shfl_xor(out[u], x, 64);
        if ((t & 63) < 8) *(v4f*)&part[i & 1][wave][4 * (t & 7)] = out;
        __syncthreads();                      // one a token: the next token writes the other half
        if (t < 8 && mine) {
            const v4f sum = (*(const v4f*)&part[i & 1][0][4 * t] + *(const v4f*)&part[i & 1][1][4 * t]) +
                            (*(const v4f*)&part[i & 1][2][4 * t] + *(const v4f*)&part[i & 1][3][4 * t]);
            *(v4f*)(y + (size_t)i * p.y.l + col) = sum * p.scale;
        }
    }
    if (t < 8 && mine)
        for (int i = len; i < p.L; i++) *(v4f*)(y + (size_t)i * p.y.l + col) = (v4f)(0.0f);
    if (p.last && mine) {
#pragma unroll
        for (int a = 0; a < STEP_ROWS; a++) {
            const int row = row0 + 32 * a;
            if (row < p.dk) *(v4f*)(p.last + base + (size_t)row * p.dv) = s[a];
        }
    }
}

// ---------------------------------------------------------------- host side
constexpr int STEPS_MAX = 16;     // up to here the recurrence

int decay_chunk(int dK4, int dV4) { return (dK4 > dV4 ? dK4 : dV4) > 64 ? 256 : 128; }

long long decay_state_bytes(int N, int head, int L, int dK4, int dV4) {
    const int C = decay_chunk(dK4, dV4);
    return (long long)N * head * ((L + C - 1) / C) * dK4 * dV4 * 4;
}

bool decay_arguments_ok(int N, int head, int L, int dK4, int dV4) {
    if (N <= 0 || head <= 0 || L <= 0 || dK4 <= 0 || dV4 <= 0 || (dK4 & 3) || (dV4 & 3) || dK4 > 128 || dV4 > 128) return false;
    const long long row = (long long)head * (dK4 > dV4 ? dK4 : dV4);
    // a tile's offsets are 32-bit bytes, positions 32-bit, a launch's workgroups 31 bits
    return L < 0x7fffff00 && row * TQ * 4 < 0x7ffffff0LL && (long long)N * head * ((L + TQ - 1LL) / TQ) < 0x7fffffffLL &&
           (long long)N * head * dK4 * dV4 / 4 < 0x7fffffffLL * 128;
}

hipError_t launch_states(hipStream_t s, const float* A, MixLayout la, int ad, const float* B, MixLayout lb, int bd, const float* g,
                         const int* lens, int N, int head, int L, int C, int back, float scale, float* U) {
    DecayStates p = {A, B, la, lb, g, lens, head, L, ad, bd, C, (L + C - 1) / C, back, scale, U, N * head};
    const dim3 grid((unsigned)((long long)N * head * p.chunks)), block(NTHREADS);
    switch (((ad > bd ? ad : bd) + 31) / 32) {
        case 1: hipLaunchKernelGGL((decay_states<1, 1>), grid, block, 0, s, p); break;
        case 2: hipLaunchKernelGGL((decay_states<2, 2>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((decay_states<4, 4>), grid, block, 0, s, p); break;
    }
    return hipGetLastError();
}

hipError_t launch_scan(hipStream_t s, float* U, const float* first, float* last, const float* g, const int* lens, int N, int head,
                       int L, int C, int back, int size) {
    DecayScan p = {U, first, last, g, lens, head, L, C, (L + C - 1) / C, back, size / 4, (long long)N * head};
    const long long items = p.nh * p.size4;
    hipLaunchKernelGGL(decay_scan, dim3((unsigned)((items + NTHREADS - 1) / NTHREADS)), dim3(NTHREADS), 0, s, p);
    return hipGetLastError();
}

template <bool ST>
hipError_t launch_mix(hipStream_t s, const DecayParams& p, int N) {
    const dim3 grid((unsigned)((long long)N * p.head * p.tiles)), block(NTHREADS);
    switch (((p.xd > p.zd ? p.xd : p.zd) + 31) / 32) {
        case 1: hipLaunchKernelGGL((decay_mix<1, 1, ST>), grid, block, 0, s, p); break;
        case 2: hipLaunchKernelGGL((decay_mix<2, 2, ST>), grid, block, 0, s, p); break;
        case 3: hipLaunchKernelGGL((decay_mix<4, 3, ST>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((decay_mix<4, 4, ST>), grid, block, 0, s, p); break;
    }
    return hipGetLastError();
}

}  // namespace
}  // namespace dragon

using namespace dragon;

extern "C" {

int64_t dragon_Cuda_linear_attention_bufsize(int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4) {
    if (!decay_arguments_ok(N, head, L, dK4, dV4)) return -1;
    return L <= STEPS_MAX ? 0 : decay_state_bytes(N, head, L, dK4, dV4);
}
int64_t dragon_Cuda_linear_attention_backward_bufsize(int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4) {
    if (!decay_arguments_ok(N, head, L, dK4, dV4)) return -1;
    return 2 * decay_state_bytes(N, head, L, dK4, dV4);
}

int dragon_Cuda_linear_attention_forward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV, int64_t dDecay,
                                         int64_t dState, int64_t dY, int64_t dStateOut, int64_t dLens, int64_t dBuf,
                                         int64_t buf_size, int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4,
                                         int32_t head_inner, float scale) {
    if (streams == nullptr || length < 1 || length > 10) return hipErrorInvalidValue;
    if (dQ == 0 || dK == 0 || dV == 0 || dDecay == 0 || dY == 0 || !mix_aligned16(dQ) || !mix_aligned16(dK) || !mix_aligned16(dV) ||
        !mix_aligned16(dY) || !mix_aligned16(dState) || !mix_aligned16(dStateOut) || (dDecay & 3) || (dLens & 3))
        return hipErrorInvalidValue;
    if (!decay_arguments_ok(N, head, L, dK4, dV4) || !(scale - scale == 0.0f)) return hipErrorInvalidValue;
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
        DecaySteps p = {Q, K, V, Y, lk, lk, lv, lv, g, lens, first, last, head, L, dK4, dV4, (dV4 + STEP_COLS - 1) / STEP_COLS, scale};
        hipLaunchKernelGGL(decay_steps, dim3((unsigned)((long long)N * head * p.slabs)), dim3(NTHREADS), 0, s, p);
        return hipGetLastError();
    }
    const int C = decay_chunk(dK4, dV4), chunks = (L + C - 1) / C;
    DecayParams p = {Q, K, V, Y, lk, lk, lv, lv, g, lens, head, L, dK4, dV4, C, chunks, 0, scale, scale, first, first == nullptr,
                     (long long)state, 0, (L + TQ - 1) / TQ, N * head};
    if (chunks > 1 || last != nullptr) {
        hipError_t e = launch_states(s, K, lk, dK4, V, lv, dV4, g, lens, N, head, L, C, 0, 1.0f, U);
        if (e == hipSuccess) e = launch_scan(s, U, first, last, g, lens, N, head, L, C, 0, (int)state);
        if (e != hipSuccess) return e;
        p.state = U; p.state_nh = (long long)chunks * state; p.state_c = (long long)state;
    }
    return launch_mix<false>(s, p, N);
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
    if (!decay_arguments_ok(N, head, L, dK4, dV4) || !(scale - scale == 0.0f)) return hipErrorInvalidValue;
    const long long need = 2 * decay_state_bytes(N, head, L, dK4, dV4);
    if (dBuf == 0 || !mix_aligned16(dBuf) || buf_size < need) return hipErrorInvalidValue;
    const float* Q = (const float*)(intptr_t)dQ; const float* K = (const float*)(intptr_t)dK; const float* V = (const float*)(intptr_t)dV;
    const float* G = (const float*)(intptr_t)dDeltaY; const float* g = (const float*)(intptr_t)dDecay;
    const float* first = (const float*)(intptr_t)dState; const float* dlast = (const float*)(intptr_t)dDeltaStateOut;
    float* gQ = (float*)(intptr_t)dDeltaQ; float* gK = (float*)(intptr_t)dDeltaK; float* gV = (float*)(intptr_t)dDeltaV;
    float* gfirst = (float*)(intptr_t)dDeltaState;
    const int* lens = (const int*)(intptr_t)dLens;
    const int C = decay_chunk(dK4, dV4), chunks = (L + C - 1) / C;
    const long long state = (long long)dK4 * dV4;
    float* S = (float*)(intptr_t)dBuf;
    float* R = S + (size_t)N * head * chunks * state;
    const MixLayout lk = mix_layout(head_inner, head, L, dK4), lv = mix_layout(head_inner, head, L, dV4);
    split_ledger_touch(gQ, (size_t)N * head * L * dK4 * 4);
    split_ledger_touch(gK, (size_t)N * head * L * dK4 * 4);
    split_ledger_touch(gV, (size_t)N * head * L * dV4 * 4);
    if (gfirst != nullptr) split_ledger_touch(gfirst, (size_t)N * head * state * 4);
    split_ledger_touch(S, (size_t)need);
    hipStream_t s = (hipStream_t)(intptr_t)streams[0];
    const bool many = chunks > 1;
    hipError_t e = hipSuccess;
    if (many) {
        e = launch_states(s, K, lk, dK4, V, lv, dV4, g, lens, N, head, L, C, 0, 1.0f, S);
        if (e == hipSuccess) e = launch_scan(s, S, first, nullptr, g, lens, N, head, L, C, 0, (int)state);
    }
    const bool later = many || gfirst != nullptr;
    if (later) {
        if (e == hipSuccess) e = launch_states(s, Q, lk, dK4, G, lv, dV4, g, lens, N, head, L, C, 1, scale, R);
        if (e == hipSuccess) e = launch_scan(s, R, dlast, gfirst, g, lens, N, head, L, C, 1, (int)state);
    }
    if (e != hipSuccess) return e;
    DecayParams p = {G, V, K, gQ, lv, lv, lk, lk, g, lens, head, L, dV4, dK4, C, chunks, 0, scale, scale,
                     many ? S : first, first == nullptr, many ? chunks * state : state, many ? state : 0, (L + TQ - 1) / TQ, N * head};
    e = launch_mix<true>(s, p, N);
    p.back = 1; p.far_scale = 1.0f;
    p.state = later ? R : dlast; p.empty_first = dlast == nullptr;
    p.state_nh = later ? chunks * state : state; p.state_c = later ? state : 0;
    p.x = V; p.y = G; p.z = Q; p.out = gK;
    if (e == hipSuccess) e = launch_mix<true>(s, p, N);
    p.x = K; p.y = Q; p.z = G; p.out = gV; p.lx = p.ly = lk; p.lz = p.lo = lv; p.xd = dK4; p.zd = dV4;
    if (e == hipSuccess) e = launch_mix<false>(s, p, N);
    return e;
}

}  // extern "C"
