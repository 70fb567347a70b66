// Selective state space memory: the short causal convolution, the scan, their backward passes and their single-token
// forms.  Rows are (sequence, time step), features are contiguous; states, statistics and parameter gradients are
// float32 whatever the sequences' type.
#include "vsv_ops.h"

namespace vsv {
namespace {

constexpr int kConvChunk = 32;       // time steps per thread of the convolution

__device__ inline long seq_len(const int* lengths, long b, long T) {
    if (!lengths) return T;
    const long n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}

// ---- short causal convolution ------------------------------------------------------------------------------------
// One output from the window, tap by tap and each operation rounded by itself: a prompt and the tokens behind it come out
// bit for bit the same, whichever kernel computes them, and so does any evaluation that takes the formula at its word -- what
// is rounded to 16 bits here feeds a recurrent state.  The exponential and the division are the accurate ones; the kernels
// wait for memory all the same.
template <int K>
__device__ inline float conv_out(const float (&w)[K], const float (&x)[K], float bias, int silu) {
#pragma clang fp contract(off)
    float s = w[0] * x[0];
#pragma unroll
    for (int k = 1; k < K; ++k) s = s + w[k] * x[k];
    s = s + bias;
    return silu ? s * (1.0f / (1.0f + expf(-s))) : s;
}

// pre[t,d] = bias[d] + sum_k w[d,k] xs[t-K+1+k, d],  y = silu(pre) or pre; xs is x, continued into state_in before t = 0.
// One read of x and one write of y (2K flops an element): bound by memory.  A thread owns VEC neighbouring channels and a
// chunk of time, so the window stays in registers and only K-1 rows per chunk are read twice.
template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) short_conv_kernel(const vsv_short_conv_desc a, long n_chunk, long n_vec) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.B * n_chunk * n_vec) return;
    const long dv = id % n_vec, bc = id / n_vec, ch = bc % n_chunk, b = bc / n_chunk;
    const long d0 = dv * VEC, t0 = ch * kConvChunk;
    const long len = seq_len(a.lengths, b, a.T);
    const long t1 = t0 + kConvChunk < a.T ? t0 + kConvChunk : a.T;
    const T* x = (const T*)a.x + b * a.x_bs + d0;
    T* y = (T*)a.y + b * a.T * a.D + d0;
    const float* st = a.state_in ? a.state_in + b * (K - 1) * a.D + d0 : nullptr;
    float w[K][VEC], bias[VEC], win[K][VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        bias[v] = a.bias ? a.bias[d0 + v] : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][v] = a.w[(d0 + v) * K + k];
    }
    auto row = [&](long t, float (&out)[VEC]) {                           // xs[t], t < len
        if (t >= 0) { load_vec<T, VEC>(x + t * a.x_ts, out); return; }
#pragma unroll
        for (int v = 0; v < VEC; ++v) out[v] = st ? st[(t + K - 1) * a.D + v] : 0.0f;
    };
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        if (t0 - K + 1 + k < len) row(t0 - K + 1 + k, win[k]);
        else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) win[k][v] = 0.0f;
        }
    }
    for (long t = t0; t < t1; ++t) {
        float out[VEC];
        if (t < len) {
            row(t, win[K - 1]);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float wv[K], xv[K];
#pragma unroll
                for (int k = 0; k < K; ++k) { wv[k] = w[k][v]; xv[k] = win[k][v]; }
                out[v] = conv_out<K>(wv, xv, bias[v], a.silu);
#pragma unroll
                for (int k = 0; k < K - 1; ++k) win[k][v] = win[k + 1][v];
            }
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) out[v] = 0.0f;
        }
        store_vec<T, VEC>(y + t * a.D, out);
    }
    if (a.state_out && ch == 0) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            float r[VEC];
            row(len - (K - 1) + j, r);
#pragma unroll
            for (int v = 0; v < VEC; ++v) a.state_out[(b * (K - 1) + j) * a.D + d0 + v] = r[v];
        }
    }
}

// ds = dy act'(pre) (pre computed again from x), dx[t] = sum_k w[k] ds[t+K-1-k], dw[k] = sum_t ds[t] xs[t-K+1+k],
// dbias = sum_t ds.  The same chunks; a chunk reads K-1 rows beyond each end, its sums over time go to `part`
// (chunk, K + 1, D) and are joined in a fixed order by sum_rows_kernel.
template <typename T, int K, int VEC>
__global__ void __launch_bounds__(256) short_conv_bwd_kernel(const vsv_short_conv_desc a, const vsv_short_conv_grads g, long n_chunk,
                                                             long n_vec, float* __restrict__ part) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.B * n_chunk * n_vec) return;
    const long dv = id % n_vec, bc = id / n_vec, ch = bc % n_chunk, b = bc / n_chunk;
    const long d0 = dv * VEC, t0 = ch * kConvChunk;
    const long len = seq_len(a.lengths, b, a.T);
    const long t1 = t0 + kConvChunk < a.T ? t0 + kConvChunk : a.T;
    const T* x = (const T*)a.x + b * a.x_bs + d0;
    const T* dy = (const T*)g.dy + b * g.dy_bs + d0;
    T* dx = (T*)g.dx + b * a.T * a.D + d0;
    const float* st = a.state_in ? a.state_in + b * (K - 1) * a.D + d0 : nullptr;
    const float* dso = g.d_state_out ? g.d_state_out + b * (K - 1) * a.D + d0 : nullptr;
    float w[K][VEC], bias[VEC], win[K][VEC], dsw[K][VEC], dw[K][VEC], db[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        bias[v] = a.bias ? a.bias[d0 + v] : 0.0f;
        db[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) { w[k][v] = a.w[(d0 + v) * K + k]; dsw[k][v] = 0.0f; dw[k][v] = 0.0f; }
    }
    auto row = [&](long t, float (&out)[VEC]) {
        if (t >= 0) { load_vec<T, VEC>(x + t * a.x_ts, out); return; }
#pragma unroll
        for (int v = 0; v < VEC; ++v) out[v] = st ? st[(t + K - 1) * a.D + v] : 0.0f;
    };
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        if (t0 - K + 1 + k < len) row(t0 - K + 1 + k, win[k]);
        else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) win[k][v] = 0.0f;
        }
    }
    const long lo = ch == 0 ? -(K - 1) : t0;                              // (chunk 0 also returns the state's gradient)
    for (long t = t0; t < t1 + K - 1; ++t) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) dsw[k][v] = dsw[k + 1][v];      // dsw[K-1-k] = ds[t-k]
        if (t < len) {
            float dyv[VEC];
            row(t, win[K - 1]);
            load_vec<T, VEC>(dy + t * g.dy_ts, dyv);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float ds = dyv[v];
                if (a.silu) {
                    float s = bias[v];
#pragma unroll
                    for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][v], win[k][v], s);
                    const float sg = sigmoid_f(s);
                    ds *= sg * (1.0f + s * (1.0f - sg));
                }
                dsw[K - 1][v] = ds;
                if (t < t1) {
                    db[v] += ds;
#pragma unroll
                    for (int k = 0; k < K; ++k) dw[k][v] = __builtin_fmaf(ds, win[k][v], dw[k][v]);
                }
#pragma unroll
                for (int k = 0; k < K - 1; ++k) win[k][v] = win[k + 1][v];
            }
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) dsw[K - 1][v] = 0.0f;
        }
        const long to = t - (K - 1);
        if (to < lo) continue;
        float o[VEC];
        const long j = to - (len - (K - 1));                              // the row of state_out that xs[to] is, if any
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][v], dsw[K - 1 - k][v], s);
            if (dso && j >= 0 && j < K - 1) s += dso[j * a.D + v];
            o[v] = s;
        }
        if (to >= 0) store_vec<T, VEC>(dx + to * a.D, o);
        else if (g.d_state_in) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) g.d_state_in[(b * (K - 1) + to + K - 1) * a.D + d0 + v] = o[v];
        }
    }
    float* p = part + (b * n_chunk + ch) * (K + 1) * a.D + d0;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
#pragma unroll
        for (int k = 0; k < K; ++k) p[k * a.D + v] = dw[k][v];
        p[(long)K * a.D + v] = db[v];
    }
}

// out_j = sum over rows of part (rows, M); element m = k * D + d goes to dw[d * K + k] or, k == K, to dbias[d].
__global__ void __launch_bounds__(256) sum_conv_parts_kernel(const float* __restrict__ part, long rows, long D, int K,
                                                             float* __restrict__ dw, float* __restrict__ dbias) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long M = (K + 1) * D, m = (long)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (m < M)
        for (long r = wave; r < rows; r += 4) s += part[r * M + m];
    red[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && m < M) {
        s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
        const long k = m / D, d = m - k * D;
        if (k < K) { if (dw) dw[d * K + k] = s; }
        else if (dbias) dbias[d] = s;
    }
}

template <typename T, int K>
__global__ void __launch_bounds__(256) short_conv_step_kernel(const T* __restrict__ x, long x_bs, float* __restrict__ state,
                                                              const float* __restrict__ w, const float* __restrict__ bias,
                                                              int silu, long B, long D, T* __restrict__ y) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= B * D) return;
    const long b = id / D, d = id - b * D;
    float win[K];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) win[k] = state[(b * (K - 1) + k) * D + d];
    win[K - 1] = to_f(x[b * x_bs + d]);
    float wv[K];
#pragma unroll
    for (int k = 0; k < K; ++k) wv[k] = w[d * K + k];
    y[b * D + d] = from_f<T>(conv_out<K>(wv, win, bias ? bias[d] : 0.0f, silu));
#pragma unroll
    for (int k = 0; k < K - 1; ++k) state[(b * (K - 1) + k) * D + d] = win[k + 1];
}

// ---- selective scan ----------------------------------------------------------------------------------------------
// delta = softplus(dt + dt_bias),  h_t = exp(delta a) h_{t-1} + delta x b_t,  y = (c_t . h_t + skip x) silu(gate).
// A lane owns a channel and its N states (padded to R), a wave 64 channels of one group, whose b_t and c_t are uniform.
constexpr int kSaveEvery = 8;        // training keeps the state before every kSaveEvery-th step

struct ScanPos { long b; long g; long d; bool live; };

__device__ inline ScanPos scan_pos(const vsv_ssm_desc& a, long blk) {
    const long Dg = a.D / a.G, cb = (Dg + 63) / 64;
    const long c = blk % cb, bg = blk / cb;
    ScanPos p;
    p.g = bg % a.G;
    p.b = bg / a.G;
    long o = c * 64 + threadIdx.x;
    p.live = o < Dg;
    if (!p.live) o = Dg - 1;
    p.d = p.g * Dg + o;
    return p;
}

template <typename T, int R>
__global__ void __launch_bounds__(64) ssm_scan_kernel(const vsv_ssm_desc a) {
    const ScanPos p = scan_pos(a, blockIdx.x);
    const long len = seq_len(a.lengths, p.b, a.T), d = p.d, D = a.D;
    const int N = a.N;
    const T *x = (const T*)a.x + p.b * a.x_bs + d, *dt = (const T*)a.dt + p.b * a.dt_bs + d;
    const T *gate = a.gate ? (const T*)a.gate + p.b * a.gate_bs + d : nullptr;
    const T *bp = (const T*)a.b + p.b * a.b_bs + p.g * a.b_gs, *cp = (const T*)a.c + p.b * a.c_bs + p.g * a.c_gs;
    T* y = (T*)a.y + p.b * a.T * D + d;
    float A2[R], h[R];
#pragma unroll
    for (int n = 0; n < R; ++n) {
        A2[n] = n < N ? a.a[d * N + n] * kLog2e : 0.0f;
        h[n] = n < N && a.state_in ? a.state_in[(p.b * D + d) * N + n] : 0.0f;
    }
    const float skip = a.skip ? a.skip[d] : 0.0f, dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    for (long t = 0; t < len; ++t) {
        if (a.saved && t % kSaveEvery == 0 && p.live) {
            float* s = a.saved + ((p.b * ((a.T + kSaveEvery - 1) / kSaveEvery) + t / kSaveEvery) * R) * D;
#pragma unroll
            for (int n = 0; n < R; ++n) s[(long)n * D + d] = h[n];
        }
        const float xv = to_f(x[t * a.x_ts]), raw = to_f(dt[t * a.dt_ts]) + dtb;
        const float de = a.softplus ? softplus_f(raw) : raw, dx = de * xv;
        float acc = skip * xv;
#pragma unroll
        for (int n = 0; n < R; ++n) {
            const float bn = n < N ? to_f(bp[t * a.b_ts + n]) : 0.0f, cn = n < N ? to_f(cp[t * a.c_ts + n]) : 0.0f;
            h[n] = __builtin_fmaf(exp2_fast(de * A2[n]), h[n], dx * bn);
            acc = __builtin_fmaf(cn, h[n], acc);
        }
        if (gate) { const float gv = to_f(gate[t * a.gate_ts]); acc *= gv * sigmoid_f(gv); }
        if (p.live) y[t * D] = from_f<T>(acc);
    }
    if (!p.live) return;
    for (long t = len; t < a.T; ++t) y[t * D] = from_f<T>(0.0f);
    if (a.state_out)
#pragma unroll
        for (int n = 0; n < R; ++n)
            if (n < N) a.state_out[(p.b * D + d) * N + n] = h[n];
}

// Backwards from the saved states, kSaveEvery steps at a time: the states of those steps are computed again into
// registers, then q_t = c_t g_t + a_{t+1} q_{t+1} (the gradient of h_t) runs through them in reverse.
template <typename T, int R>
__global__ void __launch_bounds__(64) ssm_scan_bwd_kernel(const vsv_ssm_desc a, const vsv_ssm_grads gr, float* __restrict__ part_bc,
                                                          float* __restrict__ part_p) {
    const ScanPos p = scan_pos(a, blockIdx.x);
    const long len = seq_len(a.lengths, p.b, a.T), d = p.d, D = a.D;
    const int N = a.N;
    const T *x = (const T*)a.x + p.b * a.x_bs + d, *dt = (const T*)a.dt + p.b * a.dt_bs + d;
    const T *gate = a.gate ? (const T*)a.gate + p.b * a.gate_bs + d : nullptr;
    const T *bp = (const T*)a.b + p.b * a.b_bs + p.g * a.b_gs, *cp = (const T*)a.c + p.b * a.c_bs + p.g * a.c_gs;
    const T* dy = (const T*)gr.dy + p.b * gr.dy_bs + d;
    T *dx_o = (T*)gr.dx + p.b * a.T * D + d, *ddt_o = (T*)gr.ddt + p.b * a.T * D + d;
    T* dg_o = gate ? (T*)gr.dgate + p.b * a.T * D + d : nullptr;
    const long cb = (D / a.G + 63) / 64, blk = blockIdx.x % cb;
    float* bc = part_bc + (((blk * a.B + p.b) * a.T) * a.G + p.g) * (2 * R);
    float A2[R], q[R], dA[R];
#pragma unroll
    for (int n = 0; n < R; ++n) {
        A2[n] = n < N ? a.a[d * N + n] * kLog2e : 0.0f;
        q[n] = n < N && gr.d_state_out && p.live ? gr.d_state_out[(p.b * D + d) * N + n] : 0.0f;
        dA[n] = 0.0f;
    }
    const float skip = a.skip ? a.skip[d] : 0.0f, dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    float dskip = 0.0f, ddtb = 0.0f;
    const long n_save = (a.T + kSaveEvery - 1) / kSaveEvery;
    for (long t = len; t < a.T; ++t) {
        if (p.live) {
            dx_o[t * D] = from_f<T>(0.0f);
            ddt_o[t * D] = from_f<T>(0.0f);
            if (gate) dg_o[t * D] = from_f<T>(0.0f);
        }
        if (threadIdx.x < 2 * R) bc[t * a.G * 2 * R + threadIdx.x] = 0.0f;
    }
    for (long ck = (len + kSaveEvery - 1) / kSaveEvery - 1; ck >= 0; --ck) {
        const long t0 = ck * kSaveEvery;
        const int cnt = (int)(len - t0 < kSaveEvery ? len - t0 : kSaveEvery);
        float hs[kSaveEvery + 1][R];
        const float* s = a.saved + ((p.b * n_save + ck) * R) * D;
#pragma unroll
        for (int n = 0; n < R; ++n) hs[0][n] = s[(long)n * D + d];
#pragma unroll
        for (int i = 0; i < kSaveEvery; ++i) {
            if (i >= cnt) break;
            const long t = t0 + i;
            const float xv = to_f(x[t * a.x_ts]), raw = to_f(dt[t * a.dt_ts]) + dtb;
            const float de = a.softplus ? softplus_f(raw) : raw, dx = de * xv;
#pragma unroll
            for (int n = 0; n < R; ++n) {
                const float bn = n < N ? to_f(bp[t * a.b_ts + n]) : 0.0f;
                hs[i + 1][n] = __builtin_fmaf(exp2_fast(de * A2[n]), hs[i][n], dx * bn);
            }
        }
#pragma unroll
        for (int i = kSaveEvery - 1; i >= 0; --i) {
            if (i >= cnt) continue;
            const long t = t0 + i;
            const float xv = to_f(x[t * a.x_ts]), raw = to_f(dt[t * a.dt_ts]) + dtb;
            const float de = a.softplus ? softplus_f(raw) : raw, dx = de * xv;
            float g = p.live ? to_f(dy[t * gr.dy_ts]) : 0.0f, gv = 0.0f, sg = 0.0f, dyv = g;
            if (gate) { gv = to_f(gate[t * a.gate_ts]); sg = sigmoid_f(gv); g *= gv * sg; }
            float yv = skip * xv, qb = 0.0f, dde = 0.0f;
#pragma unroll
            for (int n = 0; n < R; ++n) {
                const float bn = n < N ? to_f(bp[t * a.b_ts + n]) : 0.0f, cn = n < N ? to_f(cp[t * a.c_ts + n]) : 0.0f;
                q[n] = __builtin_fmaf(cn, g, q[n]);
                yv = __builtin_fmaf(cn, hs[i + 1][n], yv);
                qb = __builtin_fmaf(bn, q[n], qb);
                float db = p.live ? q[n] * dx : 0.0f, dc = g * hs[i + 1][n];
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) { db += __shfl_xor(db, o, 64); dc += __shfl_xor(dc, o, 64); }
                if (threadIdx.x == 0) { bc[t * a.G * 2 * R + n] = db; bc[t * a.G * 2 * R + R + n] = dc; }
                q[n] *= exp2_fast(de * A2[n]);
                const float w = q[n] * hs[i][n];
                dde = __builtin_fmaf(A2[n], w, dde);
                dA[n] = __builtin_fmaf(de, w, dA[n]);
            }
            dde = dde * (1.0f / kLog2e) + xv * qb;
            const float draw = a.softplus ? dde * sigmoid_f(raw) : dde;
            dskip = __builtin_fmaf(g, xv, dskip);
            ddtb += draw;
            if (p.live) {
                dx_o[t * D] = from_f<T>(__builtin_fmaf(qb, de, g * skip));
                ddt_o[t * D] = from_f<T>(draw);
                if (gate) dg_o[t * D] = from_f<T>(dyv * yv * sg * (1.0f + gv * (1.0f - sg)));
            }
        }
    }
    if (!p.live) return;
    float* pp = part_p + p.b * (R + 2) * D + d;
#pragma unroll
    for (int n = 0; n < R; ++n) {
        pp[(long)n * D] = dA[n];
        if (n < N && gr.d_state_in) gr.d_state_in[(p.b * D + d) * N + n] = q[n];
    }
    pp[(long)R * D] = dskip;
    pp[(long)(R + 1) * D] = ddtb;
}

// db, dc: the channel blocks' shares (blocks, B T G, 2 R) joined in order and rounded once
template <typename T>
__global__ void __launch_bounds__(256) ssm_sum_bc_kernel(const float* __restrict__ part, long blocks, long rows, int R, int N,
                                                         T* __restrict__ db, T* __restrict__ dc) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= rows * 2 * R) return;
    const long r = id / (2 * R);
    const int j = (int)(id - r * 2 * R), n = j < R ? j : j - R;
    if (n >= N) return;
    float s = 0.0f;
    for (long k = 0; k < blocks; ++k) s += part[k * rows * 2 * R + id];
    (j < R ? db : dc)[r * N + n] = from_f<T>(s);
}

// da, dskip, d_dt_bias: the sequences' shares (rows, R + 2, D) joined in order
__global__ void __launch_bounds__(256) ssm_sum_params_kernel(const float* __restrict__ part, long rows, long D, int R, int N,
                                                             float* __restrict__ da, float* __restrict__ dskip,
                                                             float* __restrict__ ddtb) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (R + 2) * D) return;
    const long n = id / D, d = id - n * D;
    float s = 0.0f;
    for (long r = 0; r < rows; ++r) s += part[r * (R + 2) * D + id];
    if (n < N) { if (da) da[d * N + n] = s; }
    else if (n == R) { if (dskip) dskip[d] = s; }
    else if (n == R + 1) { if (ddtb) ddtb[d] = s; }
}

// One step of every row.  The state's read and write are the work: P = R/4 lanes share a channel, each moving four
// states as one access, and add up the output over the P lanes.
template <typename T, int R, bool FULL>
__global__ void __launch_bounds__(256) ssm_step_kernel(const vsv_ssm_desc a) {
    constexpr int P = R / 4;
    const long id = ((long)blockIdx.x * 256 + threadIdx.x) / P;
    const int part = threadIdx.x % P, n0 = part * 4;
    if (id >= a.B * a.D) return;                                          // (all P lanes of a channel leave together)
    const long b = id / a.D, d = id - b * a.D, g = d / (a.D / a.G);
    const int N = a.N;
    const float xv = to_f(((const T*)a.x)[b * a.x_bs + d]);
    const float raw = to_f(((const T*)a.dt)[b * a.dt_bs + d]) + (a.dt_bias ? a.dt_bias[d] : 0.0f);
    const float de = a.softplus ? softplus_f(raw) : raw, dx = de * xv;
    const T *bp = (const T*)a.b + b * a.b_bs + g * a.b_gs, *cp = (const T*)a.c + b * a.c_bs + g * a.c_gs;
    float* st = a.state_out + id * N + n0;
    const float* ap = a.a + d * N + n0;
    float h[4] = {}, av[4] = {}, acc = 0.0f;
    if (FULL) { load_vec<float, 4>(st, h); load_vec<float, 4>(ap, av); }
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < N) { h[j] = st[j]; av[j] = ap[j]; }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (!FULL && n0 + j >= N) continue;
        h[j] = __builtin_fmaf(exp2_fast(de * av[j] * kLog2e), h[j], dx * to_f(bp[n0 + j]));
        acc = __builtin_fmaf(to_f(cp[n0 + j]), h[j], acc);
    }
    if (FULL) store_vec<float, 4>(st, h);
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < N) st[j] = h[j];
    }
#pragma unroll
    for (int o = 1; o < P; o <<= 1) acc += __shfl_xor(acc, o, 64);
    if (part) return;
    if (a.skip) acc = __builtin_fmaf(a.skip[d], xv, acc);
    if (a.gate) { const float gv = to_f(((const T*)a.gate)[b * a.gate_bs + d]); acc *= gv * sigmoid_f(gv); }
    ((T*)a.y)[id] = from_f<T>(acc);
}

// ---- launchers ---------------------------------------------------------------------------------------------------
constexpr long kMaxBlocks = 0x7fffffffL;

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_conv(const vsv_short_conv_desc* a, const char* what) {
    if (!a) { set_error("%s: null descriptor", what); return -1; }
    if (a->K < 1 || a->K > VSV_CONV_MAX_TAPS) { set_error("%s: %d taps; 1 to %d are built", what, a->K, VSV_CONV_MAX_TAPS); return -1; }
    if (a->B < 0 || a->T < 0 || a->D < 1) { set_error("%s: bad sizes (B %ld, T %ld, D %ld)", what, a->B, a->T, a->D); return -1; }
    if (a->dtype < VSV_F32 || a->dtype > VSV_F16) { set_error("%s: dtype must be VSV_F32, VSV_BF16 or VSV_F16", what); return -1; }
    if (!a->w || (a->B > 0 && a->T > 0 && (!a->x || !a->y))) { set_error("%s: null pointer", what); return -1; }
    return 0;
}

// 16 bytes per access where every row starts on them
bool conv_wide(const vsv_short_conv_desc* a, const vsv_short_conv_grads* g, size_t size, long vec) {
    bool ok = a->D % vec == 0 && a->x_bs % vec == 0 && a->x_ts % vec == 0 && aligned(a->x, vec * size) && aligned(a->y, vec * size);
    if (g) ok = ok && g->dy_bs % vec == 0 && g->dy_ts % vec == 0 && aligned(g->dy, vec * size) && aligned(g->dx, vec * size);
    return ok;
}

long conv_chunks(const vsv_short_conv_desc* a) { return a->T > 0 ? (a->T + kConvChunk - 1) / kConvChunk : 1; }

template <typename F> int by_taps(int K, F&& f) {
    switch (K) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        default: return f(std::integral_constant<int, 4>{});
    }
}

int check_ssm(const vsv_ssm_desc* a, const char* what) {
    if (!a) { set_error("%s: null descriptor", what); return -1; }
    if (a->N < 1 || a->N > VSV_SSM_MAX_STATE) { set_error("%s: %d states per channel; 1 to %d are built", what, a->N, VSV_SSM_MAX_STATE); return -1; }
    if (a->B < 0 || a->T < 0 || a->D < 1) { set_error("%s: bad sizes (B %ld, T %ld, D %ld)", what, a->B, a->T, a->D); return -1; }
    if (a->G < 1 || a->D % a->G) { set_error("%s: %ld channels do not divide into %ld groups", what, a->D, a->G); return -1; }
    if (a->dtype < VSV_F32 || a->dtype > VSV_F16) { set_error("%s: dtype must be VSV_F32, VSV_BF16 or VSV_F16", what); return -1; }
    if (!a->a || (a->B > 0 && a->T > 0 && (!a->x || !a->dt || !a->b || !a->c || !a->y))) { set_error("%s: null pointer", what); return -1; }
    return 0;
}

int padded_states(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : 16; }

template <typename F> int by_states(int N, F&& f) {
    switch (padded_states(N)) {
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        default: return f(std::integral_constant<int, 16>{});
    }
}

long ssm_blocks(const vsv_ssm_desc* a) { return (a->D / a->G + 63) / 64; }

}  // namespace
}  // namespace vsv

using namespace vsv;

extern "C" int vsv_short_conv(const vsv_short_conv_desc* a, void* stream) {
    if (int rc = check_conv(a, "vsv_short_conv")) return rc;
    if (a->B == 0) return 0;
    return by_dtype(a->dtype, "vsv_short_conv", [&](auto t) {
        using T = decltype(t);
        return by_taps(a->K, [&](auto k) {
            constexpr int K = decltype(k)::value, V = 16 / sizeof(T);
            const bool wide = conv_wide(a, nullptr, sizeof(T), V);
            const long nc = conv_chunks(a), nv = wide ? a->D / V : a->D, blocks = (a->B * nc * nv + 255) / 256;
            if (blocks > kMaxBlocks) { set_error("vsv_short_conv: too many elements for one call"); return -2; }
            if (wide) hipLaunchKernelGGL((short_conv_kernel<T, K, V>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, nc, nv);
            else hipLaunchKernelGGL((short_conv_kernel<T, K, 1>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, nc, nv);
            return op_launch_check("short_conv_kernel");
        });
    });
}

extern "C" size_t vsv_short_conv_backward_ws_bytes(const vsv_short_conv_desc* a) {
    if (check_conv(a, "vsv_short_conv_backward_ws_bytes")) return 0;
    return (size_t)a->B * conv_chunks(a) * (a->K + 1) * a->D * sizeof(float);
}

extern "C" int vsv_short_conv_backward(const vsv_short_conv_desc* a, const vsv_short_conv_grads* g, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_conv(a, "vsv_short_conv_backward")) return rc;
    if (!g || (a->B > 0 && a->T > 0 && (!g->dy || !g->dx))) { set_error("vsv_short_conv_backward: null pointer"); return -1; }
    if (ws_bytes < vsv_short_conv_backward_ws_bytes(a) || (!ws && a->B > 0)) { set_error("vsv_short_conv_backward: workspace too small"); return -1; }
    const long nc = conv_chunks(a), M = (a->K + 1) * a->D;
    if (a->B > 0) {
        const int rc = by_dtype(a->dtype, "vsv_short_conv_backward", [&](auto t) {
            using T = decltype(t);
            return by_taps(a->K, [&](auto k) {
                constexpr int K = decltype(k)::value, V = 16 / sizeof(T);
                const bool wide = conv_wide(a, g, sizeof(T), V);
                const long nv = wide ? a->D / V : a->D, blocks = (a->B * nc * nv + 255) / 256;
                if (blocks > kMaxBlocks) { set_error("vsv_short_conv_backward: too many elements for one call"); return -2; }
                if (wide) hipLaunchKernelGGL((short_conv_bwd_kernel<T, K, V>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, *g, nc, nv, (float*)ws);
                else hipLaunchKernelGGL((short_conv_bwd_kernel<T, K, 1>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, *g, nc, nv, (float*)ws);
                return op_launch_check("short_conv_bwd_kernel");
            });
        });
        if (rc) return rc;
    }
    hipLaunchKernelGGL(sum_conv_parts_kernel, dim3((unsigned)((M + 63) / 64)), dim3(256), 0, (hipStream_t)stream, (const float*)ws, a->B * nc, a->D, a->K, g->dw, g->dbias);
    return op_launch_check("sum_conv_parts_kernel");
}

extern "C" int vsv_short_conv_step(const vsv_short_conv_desc* a, void* stream) {
    if (int rc = check_conv(a, "vsv_short_conv_step")) return rc;
    if (a->B == 0) return 0;
    if (!a->x || !a->y || (a->K > 1 && !a->state_out)) { set_error("vsv_short_conv_step: null pointer"); return -1; }
    const long blocks = (a->B * a->D + 255) / 256;
    if (blocks > kMaxBlocks) { set_error("vsv_short_conv_step: too many elements for one call"); return -2; }
    return by_dtype(a->dtype, "vsv_short_conv_step", [&](auto t) {
        using T = decltype(t);
        return by_taps(a->K, [&](auto k) {
            hipLaunchKernelGGL((short_conv_step_kernel<T, decltype(k)::value>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                               (const T*)a->x, a->x_bs, a->state_out, a->w, a->bias, a->silu, a->B, a->D, (T*)a->y);
            return op_launch_check("short_conv_step_kernel");
        });
    });
}

extern "C" size_t vsv_ssm_saved_floats(const vsv_ssm_desc* a) {
    if (check_ssm(a, "vsv_ssm_saved_floats")) return 0;
    return (size_t)a->B * ((a->T + kSaveEvery - 1) / kSaveEvery) * padded_states(a->N) * a->D;
}

extern "C" size_t vsv_ssm_scan_ws_bytes(const vsv_ssm_desc* a) {
    if (check_ssm(a, "vsv_ssm_scan_ws_bytes")) return 0;
    return 0;
}

extern "C" int vsv_ssm_scan(const vsv_ssm_desc* a, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_ssm(a, "vsv_ssm_scan")) return rc;
    (void)ws; (void)ws_bytes;
    if (a->B == 0) return 0;
    const long blocks = a->B * a->G * ssm_blocks(a);
    if (blocks > kMaxBlocks) { set_error("vsv_ssm_scan: too many sequences and channels for one call"); return -2; }
    return by_dtype(a->dtype, "vsv_ssm_scan", [&](auto t) {
        using T = decltype(t);
        return by_states(a->N, [&](auto r) {
            hipLaunchKernelGGL((ssm_scan_kernel<T, decltype(r)::value>), dim3((unsigned)blocks), dim3(64), 0, (hipStream_t)stream, *a);
            return op_launch_check("ssm_scan_kernel");
        });
    });
}

extern "C" size_t vsv_ssm_scan_backward_ws_bytes(const vsv_ssm_desc* a) {
    if (check_ssm(a, "vsv_ssm_scan_backward_ws_bytes")) return 0;
    const size_t R = padded_states(a->N);
    return ((size_t)ssm_blocks(a) * a->B * a->T * a->G * 2 * R + (size_t)a->B * (R + 2) * a->D) * sizeof(float);
}

extern "C" int vsv_ssm_scan_backward(const vsv_ssm_desc* a, const vsv_ssm_grads* g, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_ssm(a, "vsv_ssm_scan_backward")) return rc;
    if (!g || (a->B > 0 && a->T > 0 && (!a->saved || !g->dy || !g->dx || !g->ddt || !g->db || !g->dc || (a->gate && !g->dgate)))) {
        set_error("vsv_ssm_scan_backward: null pointer"); return -1;
    }
    if (ws_bytes < vsv_ssm_scan_backward_ws_bytes(a) || (!ws && a->B > 0)) { set_error("vsv_ssm_scan_backward: workspace too small"); return -1; }
    const long nb = ssm_blocks(a), blocks = a->B * a->G * nb, rows = a->B * a->T * a->G;
    const int R = padded_states(a->N);
    if (blocks > kMaxBlocks || (rows * 2 * R + 255) / 256 > kMaxBlocks) { set_error("vsv_ssm_scan_backward: too many elements for one call"); return -2; }
    float *pbc = (float*)ws, *pp = pbc + (size_t)nb * rows * 2 * R;
    const int rc = by_dtype(a->dtype, "vsv_ssm_scan_backward", [&](auto t) {
        using T = decltype(t);
        if (blocks > 0) {
            const int rc = by_states(a->N, [&](auto r) {
                hipLaunchKernelGGL((ssm_scan_bwd_kernel<T, decltype(r)::value>), dim3((unsigned)blocks), dim3(64), 0, (hipStream_t)stream, *a, *g, pbc, pp);
                return op_launch_check("ssm_scan_bwd_kernel");
            });
            if (rc) return rc;
        }
        if (rows == 0) return 0;
        hipLaunchKernelGGL(ssm_sum_bc_kernel<T>, dim3((unsigned)((rows * 2 * R + 255) / 256)), dim3(256), 0, (hipStream_t)stream, pbc, nb, rows, R, a->N, (T*)g->db, (T*)g->dc);
        return op_launch_check("ssm_sum_bc_kernel");
    });
    if (rc) return rc;
    hipLaunchKernelGGL(ssm_sum_params_kernel, dim3((unsigned)(((R + 2) * a->D + 255) / 256)), dim3(256), 0, (hipStream_t)stream, pp, a->B, a->D, R, a->N, g->da, g->dskip, g->ddt_bias);
    return op_launch_check("ssm_sum_params_kernel");
}

extern "C" int vsv_ssm_step(const vsv_ssm_desc* a, void* stream) {
    if (int rc = check_ssm(a, "vsv_ssm_step")) return rc;
    if (a->B == 0) return 0;
    if (!a->x || !a->dt || !a->b || !a->c || !a->y || !a->state_out) { set_error("vsv_ssm_step: null pointer"); return -1; }
    const int R = padded_states(a->N);
    const long blocks = (a->B * a->D * (R / 4) + 255) / 256;
    if (blocks > kMaxBlocks) { set_error("vsv_ssm_step: too many rows for one call"); return -2; }
    return by_dtype(a->dtype, "vsv_ssm_step", [&](auto t) {
        using T = decltype(t);
        return by_states(a->N, [&](auto r) {
            constexpr int RR = decltype(r)::value;
            if (a->N == RR && aligned(a->state_out, 16) && aligned(a->a, 16))
                hipLaunchKernelGGL((ssm_step_kernel<T, RR, true>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a);
            else
                hipLaunchKernelGGL((ssm_step_kernel<T, RR, false>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a);
            return op_launch_check("ssm_step_kernel");
        });
    });
}
