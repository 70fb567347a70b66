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
// The decay belongs to (channel, state), so there is no matrix form: per state and step one exponential and four float32
// operations, 24 cycles of a SIMD per 64 channels, against 8 bytes of traffic per channel and step in 16 bits.  Bound by
// the vector units.
//   A lane owns a channel and its N states (padded to R) in registers, a wave 64 channels of one group.  b_t and c_t are
// the same for the whole wave: they are read through the scalar cache into scalar registers and cost no vector work and
// no shared memory.  x, dt and gate of the next kTile steps are loaded while the present ones are computed; the
// activations are taken for a tile at a time.
//   A wave runs along time alone, so where sequences and channels make fewer waves than the chip has SIMDs the time axis is
// split (scan_plan).  A first pass gives every segment's state from zero and its sum of delta; the state in front of a
// segment then follows from exp(a sum delta), one step per earlier segment, at the start of the second pass.
constexpr int kTile = 8;             // steps per tile; training keeps the state before every tile

typedef const __attribute__((address_space(4))) uint32_t* ScalarU;

struct ScanPlan {
    long seg;                        // steps per segment, a multiple of kTile
    int S;                           // segments
    // b and c as the kernels read them: in place, or as float32 rows of R states that pack_bc_kernel wrote
    const void *b, *c;
    long b_bs, b_ts, b_gs, c_bs, c_ts, c_gs;
};

struct ScanPos {
    long b, g, base, t0, t1, tz;     // sequence, group, first channel; the segment's steps [t0, t1), padding [t1, tz)
    int s;
    unsigned lane;                   // channel base + lane
    bool live;
};

__device__ inline long seq_len_s(const int* lengths, long b, long T) {
    if (!lengths) return T;
    const long n = ((const __attribute__((address_space(4))) int*)(uintptr_t)lengths)[b];
    return n < 0 ? 0 : n > T ? T : n;
}

__device__ inline ScanPos scan_pos(const vsv_ssm_desc& a, const ScanPlan& pl, unsigned blk, int s0) {
    const unsigned Dg = (unsigned)(a.D / a.G), cb = (Dg + 63) / 64;
    const unsigned w = (unsigned)(a.B * a.G) * cb;
    ScanPos p;
    p.s = (int)(blk / w) + s0;
    blk %= w;
    const unsigned c = blk % cb, bg = blk / cb;
    p.g = bg % (unsigned)a.G;
    p.b = bg / (unsigned)a.G;
    p.base = p.g * Dg + c * 64;
    const unsigned left = Dg - c * 64;
    p.live = threadIdx.x < left;
    p.lane = p.live ? threadIdx.x : left - 1;
    const long len = seq_len_s(a.lengths, p.b, a.T);
    p.t0 = p.s * pl.seg;
    p.tz = p.t0 + pl.seg < a.T ? p.t0 + pl.seg : a.T;
    p.t1 = p.tz < len ? p.tz : len;
    return p;
}

// n states of b_t or c_t, uniform over the wave, as the words that scalar loads bring.  BF: pairs of bfloat16 in place, else
// float32.  Scalar loads return out of order, so a wait is for all of them: every step waits for its own rows first, then
// asks for the next step's, and computes while these are on their way (scheduling barriers keep that order).
template <int R, bool BF> struct ScalarRow {
    uint32_t w[BF ? R / 2 : R];
    __device__ inline void load(uintptr_t p) {
        const ScalarU u = (ScalarU)p;
#pragma unroll
        for (int j = 0; j < (BF ? R / 2 : R); ++j) w[j] = u[j];
    }
    __device__ inline float at(int n) const {
        if (!BF) return __builtin_bit_cast(float, w[n]);
        return __builtin_bit_cast(float, n & 1 ? w[n / 2] & 0xffff0000u : w[n / 2] << 16);
    }
};
__device__ inline void order() { __builtin_amdgcn_sched_barrier(0); }
// An empty statement that a value passes through: what is computed from it stays behind it, in its step.  (Without it the
// steps of a tile are computed side by side, and their states do not fit the registers.)
__device__ inline void pin(float& v) { asm volatile("" : "+v"(v)); }
__device__ inline void scalar_wait() { __builtin_amdgcn_s_waitcnt(0xc07f); order(); }      // lgkmcnt(0)

// kTile rows from `row` on (those behind the first `left` repeat the last) of one channel per lane; `row` is uniform
template <typename T>
__device__ inline void load_tile(const T* row, long ts, unsigned lane, int left, T (&out)[kTile]) {
#pragma unroll
    for (int i = 0; i < kTile; ++i) {
        out[i] = row[lane];
        if (i + 1 < left) row += ts;
    }
}

// The time steps and inputs of a tile; steps at t1 and beyond get delta = x = 0, which leaves every state as it is.
template <typename T>
__device__ inline void tile_steps(const T (&dr)[kTile], float dtb, int softplus, int left, float (&raw)[kTile], float (&de)[kTile]) {
#pragma unroll
    for (int i = 0; i < kTile; ++i) de[i] = raw[i] = to_f(dr[i]) + dtb;
    if (softplus) {
#pragma unroll
        for (int i = 0; i < kTile; ++i) de[i] = softplus_f(de[i]);
    }
    if (left < kTile) {
#pragma unroll
        for (int i = 0; i < kTile; ++i)
            if (i >= left) de[i] = 0.0f;
    }
}
template <typename T> __device__ inline void tile_values(const T (&r)[kTile], int left, float (&v)[kTile]) {
#pragma unroll
    for (int i = 0; i < kTile; ++i) v[i] = to_f(r[i]);
    if (left < kTile) {
#pragma unroll
        for (int i = 0; i < kTile; ++i)
            if (i >= left) v[i] = 0.0f;
    }
}
template <typename T> __device__ inline void tile_store(T* base, long D, const ScanPos& p, long t, int left, const float (&v)[kTile]) {
    if (!p.live) return;
#pragma unroll
    for (int i = 0; i < kTile; ++i)
        if (i < left) (base + (t + i) * D)[p.lane] = from_f<T>(v[i]);
}

// State sets in memory: (R/4, D, 4), so that a wave moves 1 KiB at a time.
template <int R> __device__ inline void load_states(const float* p, long D, long d, float (&v)[R]) {
#pragma unroll
    for (int k = 0; k < R / 4; ++k) {
        float q[4];
        load_vec<float, 4>(p + (k * D + d) * 4, q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * k + j] = q[j];
    }
}
template <int R> __device__ inline void store_states(float* p, long D, long d, const float (&v)[R]) {
#pragma unroll
    for (int k = 0; k < R / 4; ++k) {
        const float q[4] = {v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
        store_vec<float, 4>(p + (k * D + d) * 4, q);
    }
}

__device__ inline int tile_left(const ScanPos& p, long t) { return p.t1 - t < kTile ? (int)(p.t1 - t) : kTile; }

template <int R> __device__ inline void load_decay(const vsv_ssm_desc& a, long d, float (&A2)[R]) {
#pragma unroll
    for (int n = 0; n < R; ++n) A2[n] = n < a.N ? a.a[d * a.N + n] * kLog2e : 0.0f;
}

// v = exp(a sum delta) v + E over the segments from, from + step, .. up to (not including) to
template <int R>
__device__ inline void fold_segments(const float* E, const float* sd, long D, long d, long row0, int from, int to, int step,
                                     const float (&A2)[R], float (&v)[R]) {
    for (int k = from; k != to; k += step) {
        float e[R];
        load_states<R>(E + (row0 + k) * R * D, D, d, e);
        const float s = sd[(row0 + k) * D + d];
#pragma unroll
        for (int n = 0; n < R; ++n) v[n] = __builtin_fmaf(exp2_fast(s * A2[n]), v[n], e[n]);
    }
}

// First pass of a split scan: a segment's last state from zero, and its sum of delta.
template <typename T, int R, bool BF>
__global__ void __launch_bounds__(64) ssm_ends_kernel(const vsv_ssm_desc a, const ScanPlan pl, float* __restrict__ E, float* __restrict__ sd) {
    constexpr long kEl = BF ? 2 : 4;
    const ScanPos p = scan_pos(a, pl, blockIdx.x, 0);
    const long D = a.D, d = p.base + p.lane;
    float A2[R], h[R] = {}, sum = 0.0f;
    load_decay<R>(a, d, A2);
    const float dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    const T *x = (const T*)a.x + p.b * a.x_bs + p.base + p.t0 * a.x_ts, *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + p.t0 * a.dt_ts;
    uintptr_t pb = (uintptr_t)pl.b + (p.b * pl.b_bs + p.g * pl.b_gs + p.t0 * pl.b_ts) * kEl;
    ScalarRow<R, BF> b;
    T xr[kTile], dr[kTile];
    if (p.t0 < p.t1) {
        b.load(pb);
        load_tile(x, a.x_ts, p.lane, tile_left(p, p.t0), xr);
        load_tile(dt, a.dt_ts, p.lane, tile_left(p, p.t0), dr);
    }
    for (long t = p.t0; t < p.t1; t += kTile) {
        const int left = tile_left(p, t);
        const bool more = t + kTile < p.t1;
        float xv[kTile], raw[kTile], de[kTile];
        tile_values(xr, left, xv);
        tile_steps(dr, dtb, a.softplus, left, raw, de);
        if (more) {
            x += kTile * a.x_ts; dt += kTile * a.dt_ts;
            load_tile(x, a.x_ts, p.lane, tile_left(p, t + kTile), xr);
            load_tile(dt, a.dt_ts, p.lane, tile_left(p, t + kTile), dr);
        }
        order();
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            ScalarRow<R, BF> nb;
            scalar_wait();
            if (i + 1 < left || more) pb += pl.b_ts * kEl;
            nb.load(pb);
            order();
            const float dx = de[i] * xv[i];
            sum += de[i];
#pragma unroll
            for (int n = 0; n < R; ++n) h[n] = __builtin_fmaf(exp2_fast(de[i] * A2[n]), h[n], dx * b.at(n));
            order();
            b = nb;
        }
    }
    if (!p.live) return;
    store_states<R>(E + (p.b * pl.S + p.s) * R * D, D, d, h);
    sd[(p.b * pl.S + p.s) * D + d] = sum;
}

template <typename T, int R, bool BF>
__global__ void __launch_bounds__(64) ssm_scan_kernel(const vsv_ssm_desc a, const ScanPlan pl, const float* __restrict__ E,
                                                      const float* __restrict__ sd) {
    constexpr long kEl = BF ? 2 : 4;
    const ScanPos p = scan_pos(a, pl, blockIdx.x, 0);
    const long D = a.D, d = p.base + p.lane;
    const int N = a.N;
    T* y = (T*)a.y + p.b * a.T * D + p.base;
    float A2[R], h[R];
    load_decay<R>(a, d, A2);
#pragma unroll
    for (int n = 0; n < R; ++n) h[n] = n < N && a.state_in ? a.state_in[(p.b * D + d) * N + n] : 0.0f;
    fold_segments<R>(E, sd, D, d, p.b * pl.S, 0, p.s, 1, A2, h);
    const float skip = a.skip ? a.skip[d] : 0.0f, dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    const T *x = (const T*)a.x + p.b * a.x_bs + p.base + p.t0 * a.x_ts, *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + p.t0 * a.dt_ts;
    const T* gate = a.gate ? (const T*)a.gate + p.b * a.gate_bs + p.base + p.t0 * a.gate_ts : nullptr;
    uintptr_t pb = (uintptr_t)pl.b + (p.b * pl.b_bs + p.g * pl.b_gs + p.t0 * pl.b_ts) * kEl;
    uintptr_t pc = (uintptr_t)pl.c + (p.b * pl.c_bs + p.g * pl.c_gs + p.t0 * pl.c_ts) * kEl;
    float* saved = a.saved ? a.saved + (p.b * ((a.T + kTile - 1) / kTile) + p.t0 / kTile) * R * D : nullptr;
    ScalarRow<R, BF> b, c;
    T xr[kTile], dr[kTile], gr[kTile];
    auto fetch = [&](int left) {
        load_tile(x, a.x_ts, p.lane, left, xr);
        load_tile(dt, a.dt_ts, p.lane, left, dr);
        if (gate) load_tile(gate, a.gate_ts, p.lane, left, gr);
    };
    if (p.t0 < p.t1) { b.load(pb); c.load(pc); fetch(tile_left(p, p.t0)); }
    for (long t = p.t0; t < p.t1; t += kTile) {
        const int left = tile_left(p, t);
        const bool more = t + kTile < p.t1;
        float xv[kTile], raw[kTile], de[kTile], gv[kTile], yv[kTile];
        tile_values(xr, left, xv);
        tile_steps(dr, dtb, a.softplus, left, raw, de);
        if (gate) {
            tile_values(gr, left, gv);
#pragma unroll
            for (int i = 0; i < kTile; ++i) gv[i] *= sigmoid_f(gv[i]);
        }
        if (more) {
            x += kTile * a.x_ts; dt += kTile * a.dt_ts; gate += gate ? kTile * a.gate_ts : 0;
            fetch(tile_left(p, t + kTile));
        }
        if (saved) {
            if (p.live) store_states<R>(saved, D, d, h);
            saved += R * D;
        }
        order();
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            ScalarRow<R, BF> nb, nc;
            scalar_wait();
            if (i + 1 < left || more) { pb += pl.b_ts * kEl; pc += pl.c_ts * kEl; }
            nb.load(pb); nc.load(pc);
            order();
            const float dx = de[i] * xv[i];
            float acc = skip * xv[i];
#pragma unroll
            for (int n = 0; n < R; ++n) {
                h[n] = __builtin_fmaf(exp2_fast(de[i] * A2[n]), h[n], dx * b.at(n));
                acc = __builtin_fmaf(c.at(n), h[n], acc);
            }
            yv[i] = acc;
            order();
            b = nb; c = nc;
        }
        if (gate) {
#pragma unroll
            for (int i = 0; i < kTile; ++i) yv[i] *= gv[i];
        }
        tile_store(y, D, p, t, left, yv);
    }
    if (!p.live) return;
    for (long t = p.t0 > p.t1 ? p.t0 : p.t1; t < p.tz; ++t) (y + t * D)[p.lane] = from_f<T>(0.0f);
    if (a.state_out && p.s == pl.S - 1)
#pragma unroll
        for (int n = 0; n < R; ++n)
            if (n < N) a.state_out[(p.b * D + d) * N + n] = h[n];
}

// Backwards: g = dy silu(gate), q_t = c_t g_t + exp(delta_{t+1} a) q_{t+1} is the gradient of h_t.
// First pass of a split one: the gradient of the state in front of a segment where none comes in from behind it.
template <typename T, int R, bool BF>
__global__ void __launch_bounds__(64) ssm_bwd_ends_kernel(const vsv_ssm_desc a, const vsv_ssm_grads gr, const ScanPlan pl, float* __restrict__ E,
                                                          float* __restrict__ sd) {
    constexpr long kEl = BF ? 2 : 4;
    const ScanPos p = scan_pos(a, pl, blockIdx.x, 1);
    const long D = a.D, d = p.base + p.lane;
    float A2[R], q[R] = {}, sum = 0.0f;
    load_decay<R>(a, d, A2);
    const float dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    const long tl = p.t0 + (p.t1 - 1 - p.t0) / kTile * kTile;              // the last tile
    const T *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + tl * a.dt_ts, *dy = (const T*)gr.dy + p.b * gr.dy_bs + p.base + tl * gr.dy_ts;
    const T* gate = a.gate ? (const T*)a.gate + p.b * a.gate_bs + p.base + tl * a.gate_ts : nullptr;
    uintptr_t pc = (uintptr_t)pl.c + (p.b * pl.c_bs + p.g * pl.c_gs + (p.t1 - 1) * pl.c_ts) * kEl;
    ScalarRow<R, BF> c;
    T dr[kTile], gtr[kTile], yr[kTile];
    auto fetch = [&](int left) {
        load_tile(dt, a.dt_ts, p.lane, left, dr);
        load_tile(dy, gr.dy_ts, p.lane, left, yr);
        if (gate) load_tile(gate, a.gate_ts, p.lane, left, gtr);
    };
    if (p.t0 < p.t1) { c.load(pc); fetch(tile_left(p, tl)); }
    for (long t = tl; t >= p.t0 && p.t0 < p.t1; t -= kTile) {
        const int left = tile_left(p, t);
        const bool more = t > p.t0;
        float raw[kTile], de[kTile], g[kTile];
        tile_steps(dr, dtb, a.softplus, left, raw, de);
        tile_values(yr, left, g);
        if (gate) {
            float gv[kTile];
            tile_values(gtr, left, gv);
#pragma unroll
            for (int i = 0; i < kTile; ++i) g[i] *= gv[i] * sigmoid_f(gv[i]);
        }
        if (more) {
            dt -= kTile * a.dt_ts; dy -= kTile * gr.dy_ts; gate -= gate ? kTile * a.gate_ts : 0;
            fetch(kTile);
        }
        order();
#pragma unroll
        for (int i = kTile - 1; i >= 0; --i) {
            ScalarRow<R, BF> nc;
            scalar_wait();
            if (i < left && (i > 0 || more)) pc -= pl.c_ts * kEl;
            nc.load(pc);
            order();
            sum += de[i];
#pragma unroll
            for (int n = 0; n < R; ++n) q[n] = exp2_fast(de[i] * A2[n]) * __builtin_fmaf(c.at(n), g[i], q[n]);
            order();
            if (i < left) c = nc;
        }
    }
    if (!p.live) return;
    store_states<R>(E + (p.b * pl.S + p.s) * R * D, D, d, q);
    sd[(p.b * pl.S + p.s) * D + d] = sum;
}

// Sums of NV values over the wave's 64 lanes: at every level half of the values go to the partner lane and half come from
// it, so that 2 NV operations do what 6 NV would if each value were summed by itself.  Lane l ends up with value
// l / (64 / NV).
template <int CTRL> __device__ inline float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int CTRL, int H, int NV> __device__ inline void halve(float (&v)[NV], bool upper) {
#pragma unroll
    for (int j = 0; j < H; ++j) {
        const float keep = upper ? v[j + H] : v[j], give = upper ? v[j] : v[j + H];
        v[j] = keep + dpp<CTRL>(give);
    }
}
template <int NV> __device__ inline float wave_sums(float (&v)[NV]) {
    constexpr int kRor8 = 0x128, kHalfMirror = 0x141, kXor2 = 0x4e, kXor1 = 0xb1;
    static_assert(NV == 8 || NV == 16 || NV == 32, "");
#pragma unroll
    for (int j = 0; j < NV / 2; ++j) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v[j]), __builtin_bit_cast(unsigned, v[j + NV / 2]), false, false);
        const unsigned r0 = r[0], r1 = r[1];
        v[j] = __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
    }
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v[j]), __builtin_bit_cast(unsigned, v[j + NV / 4]), false, false);
        const unsigned r0 = r[0], r1 = r[1];
        v[j] = __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
    }
    const int l = threadIdx.x;
    if constexpr (NV >= 8) halve<kRor8, NV / 8>(v, l & 8);
    if constexpr (NV >= 16) halve<kHalfMirror, NV / 16>(v, l & 4); else v[0] += dpp<kHalfMirror>(v[0]);
    if constexpr (NV >= 32) halve<kXor2, NV / 32>(v, l & 2); else v[0] += dpp<kXor2>(v[0]);
    return v[0] + dpp<kXor1>(v[0]);
}

// A tile at a time from the state saved in front of it: its states are computed again into registers, then q runs through
// them in reverse, four states at a time so that they fit.  The gradients of b and c are sums over channels: over the
// wave's 64 here, over the channel blocks in sum_bc_kernel; those of a, skip and dt_bias sums over time: here, and over
// sequences and segments in sum_params_kernel.  All in a fixed order.
template <typename T, int R, bool BF>
__global__ void __launch_bounds__(64, 2) ssm_bwd_kernel(const vsv_ssm_desc a, const vsv_ssm_grads gr, const ScanPlan pl, const float* __restrict__ E,
                                                        const float* __restrict__ sd, float* __restrict__ part_bc, float* __restrict__ part_p) {
    constexpr long kEl = BF ? 2 : 4;
    constexpr int H = 4;
    const ScanPos p = scan_pos(a, pl, blockIdx.x, 0);
    const long D = a.D, d = p.base + p.lane;
    const int N = a.N;
    const long tl = p.t0 + (p.t1 - 1 - p.t0) / kTile * kTile;              // the last tile
    const T *x = (const T*)a.x + p.b * a.x_bs + p.base + tl * a.x_ts, *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + tl * a.dt_ts;
    const T *dy = (const T*)gr.dy + p.b * gr.dy_bs + p.base + tl * gr.dy_ts;
    const T* gate = a.gate ? (const T*)a.gate + p.b * a.gate_bs + p.base + tl * a.gate_ts : nullptr;
    const float* saved = a.saved + (p.b * ((a.T + kTile - 1) / kTile) + tl / kTile) * R * D;
    const long row = p.b * a.T * D + p.base;
    T *dx_o = (T*)gr.dx + row, *ddt_o = (T*)gr.ddt + row, *dg_o = gate ? (T*)gr.dgate + row : nullptr;
    uintptr_t pb = (uintptr_t)pl.b + (p.b * pl.b_bs + p.g * pl.b_gs + tl * pl.b_ts) * kEl;
    uintptr_t pc = (uintptr_t)pl.c + (p.b * pl.c_bs + p.g * pl.c_gs + tl * pl.c_ts) * kEl;
    const long Dg = D / a.G, blk = (p.base - p.g * Dg) / 64;
    float* bc = part_bc + (((blk * a.B + p.b) * a.T) * a.G + p.g) * (2 * R);
    const long bc_ts = a.G * 2 * R;
    float A2[R], q[R], dA[R] = {};
    load_decay<R>(a, d, A2);
#pragma unroll
    for (int n = 0; n < R; ++n) q[n] = n < N && gr.d_state_out ? gr.d_state_out[(p.b * D + d) * N + n] : 0.0f;
    fold_segments<R>(E, sd, D, d, p.b * pl.S, pl.S - 1, p.s, -1, A2, q);
    if (!p.live) {
#pragma unroll
        for (int n = 0; n < R; ++n) q[n] = 0.0f;
    }
    const float skip = a.skip ? a.skip[d] : 0.0f, dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    float dskip = 0.0f, ddtb = 0.0f;
    T xr[kTile], dr[kTile], gtr[kTile], yr[kTile];
    auto fetch = [&](int left) {
        load_tile(x, a.x_ts, p.lane, left, xr);
        load_tile(dt, a.dt_ts, p.lane, left, dr);
        load_tile(dy, gr.dy_ts, p.lane, left, yr);
        if (gate) load_tile(gate, a.gate_ts, p.lane, left, gtr);
    };
    if (p.t0 < p.t1) fetch(tile_left(p, tl));
    for (long t = tl; t >= p.t0 && p.t0 < p.t1; t -= kTile) {
        const int left = tile_left(p, t);
        float h0[R], xv[kTile], raw[kTile], de[kTile], g[kTile], dsl[kTile];
        load_states<R>(saved, D, d, h0);
        tile_values(xr, left, xv);
        tile_steps(dr, dtb, a.softplus, left, raw, de);
        tile_values(yr, left, g);
        if (!p.live) {
#pragma unroll
            for (int i = 0; i < kTile; ++i) g[i] = xv[i] = 0.0f;
        }
        if (gate) {
            float gv[kTile];
            tile_values(gtr, left, gv);
#pragma unroll
            for (int i = 0; i < kTile; ++i) {
                const float sg = sigmoid_f(gv[i]);
                dsl[i] = g[i] * sg * (1.0f + gv[i] * (1.0f - sg));
                g[i] *= gv[i] * sg;
            }
        }
        if (t > p.t0) {
            x -= kTile * a.x_ts; dt -= kTile * a.dt_ts; dy -= kTile * gr.dy_ts; gate -= gate ? kTile * a.gate_ts : 0;
            saved -= R * D;
            fetch(kTile);
        }
        float qb[kTile] = {}, dde[kTile] = {}, yv[kTile] = {};
#pragma unroll
        for (int n0 = 0; n0 < R; n0 += H) {
            float hs[kTile + 1][H];
            ScalarRow<H, BF> b, c, nb, nc;
            b.load(pb + n0 * kEl);
#pragma unroll
            for (int n = 0; n < H; ++n) hs[0][n] = h0[n0 + n];
            uintptr_t rb = pb + n0 * kEl;
            order();
#pragma unroll
            for (int i = 0; i < kTile; ++i) {
                scalar_wait();
                if (i + 1 < left) rb += pl.b_ts * kEl;
                if (i + 1 < kTile) nb.load(rb);
                else c.load(pc + (n0 + (left - 1) * pl.c_ts) * kEl);       // (b stays: the reverse starts at the same row)
                order();
                float dei = de[i];
                pin(dei);
                const float dx = dei * xv[i];
#pragma unroll
                for (int n = 0; n < H; ++n) {
                    hs[i + 1][n] = __builtin_fmaf(exp2_fast(dei * A2[n0 + n]), hs[i][n], dx * b.at(n));
                    pin(hs[i + 1][n]);
                }
                order();
                if (i + 1 < kTile) b = nb;
            }
            uintptr_t rc = pc + (n0 + (left - 1) * pl.c_ts) * kEl;
#pragma unroll
            for (int i = kTile - 1; i >= 0; --i) {
                float v[2 * H];
                scalar_wait();
                if (i > 0) {
                    if (i < left) { rb -= pl.b_ts * kEl; rc -= pl.c_ts * kEl; }
                    nb.load(rb); nc.load(rc);
                }
                order();
                float dei = de[i];
                pin(dei);
                const float dx = dei * xv[i];
#pragma unroll
                for (int n = 0; n < H; ++n) {
                    float& qn = q[n0 + n];
                    qn = __builtin_fmaf(c.at(n), g[i], qn);
                    yv[i] = __builtin_fmaf(c.at(n), hs[i + 1][n], yv[i]);
                    qb[i] = __builtin_fmaf(b.at(n), qn, qb[i]);
                    v[n] = qn * dx;
                    v[H + n] = g[i] * hs[i + 1][n];
                    qn *= exp2_fast(dei * A2[n0 + n]);
                    const float w = qn * hs[i][n];
                    dde[i] = __builtin_fmaf(A2[n0 + n], w, dde[i]);
                    dA[n0 + n] = __builtin_fmaf(dei, w, dA[n0 + n]);
                    pin(qn); pin(dA[n0 + n]);
                }
                pin(yv[i]); pin(qb[i]); pin(dde[i]);
                const float sum = wave_sums<2 * H>(v);
                constexpr int kEach = 64 / (2 * H);
                if (i < left && threadIdx.x % kEach == 0) {
                    const int j = threadIdx.x / kEach;                      // b's four states, then c's
                    bc[(t + i) * bc_ts + n0 + (j < H ? j : j - H + R)] = sum;
                }
                order();
                b = nb; c = nc;
            }
        }
        pb -= kTile * pl.b_ts * kEl; pc -= kTile * pl.c_ts * kEl;
        float dxv[kTile], ddv[kTile];
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            const float dd = __builtin_fmaf(xv[i], qb[i], dde[i] * (1.0f / kLog2e));
            ddv[i] = i < left ? (a.softplus ? dd * sigmoid_f(raw[i]) : dd) : 0.0f;
            dskip = __builtin_fmaf(g[i], xv[i], dskip);
            ddtb += ddv[i];
            dxv[i] = __builtin_fmaf(qb[i], de[i], g[i] * skip);
        }
        tile_store(dx_o, D, p, t, left, dxv);
        tile_store(ddt_o, D, p, t, left, ddv);
        if (gate) {
#pragma unroll
            for (int i = 0; i < kTile; ++i) yv[i] = dsl[i] * __builtin_fmaf(skip, xv[i], yv[i]);
            tile_store(dg_o, D, p, t, left, yv);
        }
    }
    for (long t = p.t0 > p.t1 ? p.t0 : p.t1; t < p.tz; ++t) {
        if (p.live) {
            (dx_o + t * D)[p.lane] = from_f<T>(0.0f);
            (ddt_o + t * D)[p.lane] = from_f<T>(0.0f);
            if (gate) (dg_o + t * D)[p.lane] = from_f<T>(0.0f);
        }
        if (threadIdx.x < 2 * R) bc[t * bc_ts + threadIdx.x] = 0.0f;
    }
    if (!p.live) return;
    float* pp = part_p + (p.b * pl.S + p.s) * (R + 2) * D + d;
#pragma unroll
    for (int n = 0; n < R; ++n) pp[(long)n * D] = dA[n];
    pp[(long)R * D] = dskip;
    pp[(long)(R + 1) * D] = ddtb;
    if (gr.d_state_in && p.s == 0)
#pragma unroll
        for (int n = 0; n < R; ++n)
            if (n < N) gr.d_state_in[(p.b * D + d) * N + n] = q[n];
}

// b and c (any strides, N states) as float32 rows (B, T, G, 2, R), padded with zeros: what the scalar loads need where the
// tensors themselves are not whole, aligned words.
template <typename T>
__global__ void __launch_bounds__(256) pack_bc_kernel(const vsv_ssm_desc a, int R, float* __restrict__ out) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.B * a.T * a.G * 2 * R) return;
    const int j = (int)(id % (2 * R)), n = j < R ? j : j - R;
    const long r = id / (2 * R), g = r % a.G, bt = r / a.G, t = bt % a.T, b = bt / a.T;
    float v = 0.0f;
    if (n < a.N)
        v = to_f(j < R ? ((const T*)a.b)[b * a.b_bs + t * a.b_ts + g * a.b_gs + n] : ((const T*)a.c)[b * a.c_bs + t * a.c_ts + g * a.c_gs + n]);
    out[id] = v;
}

// db, dc: the channel blocks' shares (blocks, B T G, 2 R) joined in order and rounded once
template <typename T>
__global__ void __launch_bounds__(256) sum_bc_kernel(const float* __restrict__ part, long blocks, long rows, int R, int N,
                                                     T* __restrict__ db, T* __restrict__ dc) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x, M = rows * 2 * R;
    if (id >= M) return;
    const long r = id / (2 * R);
    const int j = (int)(id - r * 2 * R), n = j < R ? j : j - R;
    if (n >= N) return;
    float s = 0.0f;
#pragma unroll 8
    for (long k = 0; k < blocks; ++k) s += part[k * M + id];
    (j < R ? db : dc)[r * N + n] = from_f<T>(s);
}

// da, dskip, d_dt_bias: the sequences' and segments' shares (rows, R + 2, D) joined in order
__global__ void __launch_bounds__(256) sum_params_kernel(const float* __restrict__ part, long rows, long D, int R, int N,
                                                         float* __restrict__ da, float* __restrict__ dskip, float* __restrict__ ddtb) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long M = (R + 2) * D, m = (long)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (m < M) {
#pragma unroll 8
        for (long r = wave; r < rows; r += 4) s += part[r * M + m];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave || m >= M) return;
    s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    const long n = m / D, d = m - n * D;
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

// The scan's split of time.  A second pass over a segment costs 1.8 times one pass over it, so a split pays below about
// half a wave per SIMD (1024 of them): from there on as many segments as make two waves per SIMD, none shorter than two
// tiles, at most kMaxSegments (the start of a segment walks over those in front of it).
constexpr long kMaxSegments = 64;

ScanPlan scan_plan(const vsv_ssm_desc* a) {
    ScanPlan pl = {};
    const long waves = a->B * a->G * ssm_blocks(a), tiles = (a->T + kTile - 1) / kTile;
    long S = 1;
    if (waves > 0 && waves < 512 && tiles >= 4) {
        S = (2048 + waves - 1) / waves;
        if (S > tiles / 2) S = tiles / 2;
        if (S > kMaxSegments) S = kMaxSegments;
    }
    const long per = tiles > 0 ? (tiles + S - 1) / S : 1;
    pl.seg = per * kTile;
    pl.S = tiles > 0 ? (int)((tiles + per - 1) / per) : 1;
    return pl;
}

// Whether scalar loads can read b and c in place: whole rows of R states in float32, or in bfloat16 on 4 bytes.
bool bc_in_place(const vsv_ssm_desc* a) {
    if (a->N != padded_states(a->N)) return false;
    if (a->dtype == VSV_F32) return true;
    return a->dtype == VSV_BF16 && aligned(a->b, 4) && aligned(a->c, 4) &&
           ((a->b_bs | a->b_ts | a->b_gs | a->c_bs | a->c_ts | a->c_gs) & 1) == 0;
}

size_t bc_floats(const vsv_ssm_desc* a) { return bc_in_place(a) ? 0 : (size_t)a->B * a->T * a->G * 2 * padded_states(a->N); }
size_t ends_floats(const vsv_ssm_desc* a, const ScanPlan& pl) {
    return pl.S > 1 ? (size_t)a->B * pl.S * (padded_states(a->N) + 1) * a->D : 0;
}
size_t round4(size_t n) { return (n + 3) & ~(size_t)3; }

// Points the plan at b and c, packing them into `out` first where they cannot be read in place.
template <typename T> int place_bc(const vsv_ssm_desc* a, ScanPlan& pl, float* out, void* stream, const char* what) {
    if (bc_in_place(a)) {
        pl.b = a->b; pl.b_bs = a->b_bs; pl.b_ts = a->b_ts; pl.b_gs = a->b_gs;
        pl.c = a->c; pl.c_bs = a->c_bs; pl.c_ts = a->c_ts; pl.c_gs = a->c_gs;
        return 0;
    }
    const int R = padded_states(a->N);
    pl.b = out; pl.c = out + R;
    pl.b_gs = pl.c_gs = 2 * R;
    pl.b_ts = pl.c_ts = a->G * 2 * R;
    pl.b_bs = pl.c_bs = a->T * a->G * 2 * R;
    const long blocks = ((long)bc_floats(a) + 255) / 256;
    if (blocks == 0) return 0;
    if (blocks > kMaxBlocks) { set_error("%s: too many elements for one call", what); return -2; }
    hipLaunchKernelGGL(pack_bc_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, R, out);
    return op_launch_check("pack_bc_kernel");
}

// f(T, R, whether b and c are pairs of bfloat16 in place)
template <typename F> int by_scan(const vsv_ssm_desc* a, const char* what, F&& f) {
    return by_dtype(a->dtype, what, [&](auto t) {
        return by_states(a->N, [&](auto r) {
            if constexpr (std::is_same<decltype(t), __bf16>::value) {
                if (bc_in_place(a)) return f(t, r, std::true_type{});
            }
            return f(t, r, std::false_type{});
        });
    });
}

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
    return (size_t)a->B * ((a->T + kTile - 1) / kTile) * padded_states(a->N) * a->D;
}

extern "C" size_t vsv_ssm_scan_ws_bytes(const vsv_ssm_desc* a) {
    if (check_ssm(a, "vsv_ssm_scan_ws_bytes")) return 0;
    return (round4(bc_floats(a)) + ends_floats(a, scan_plan(a))) * sizeof(float);
}

extern "C" int vsv_ssm_scan(const vsv_ssm_desc* a, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_ssm(a, "vsv_ssm_scan")) return rc;
    if (a->B == 0) return 0;
    const size_t need = vsv_ssm_scan_ws_bytes(a);
    if (ws_bytes < need || (need && !aligned(ws, 16)) || (need && !ws)) { set_error("vsv_ssm_scan: workspace too small or not on 16 bytes"); return -1; }
    if (a->saved && !aligned(a->saved, 16)) { set_error("vsv_ssm_scan: saved must be on 16 bytes"); return -1; }
    ScanPlan pl = scan_plan(a);
    const long waves = a->B * a->G * ssm_blocks(a);
    if (waves * pl.S > kMaxBlocks) { set_error("vsv_ssm_scan: too many sequences and channels for one call"); return -2; }
    float *bc = (float*)ws, *E = bc + round4(bc_floats(a)), *sd = E + (size_t)a->B * pl.S * padded_states(a->N) * a->D;
    return by_scan(a, "vsv_ssm_scan", [&](auto t, auto r, auto bf) {
        using T = decltype(t);
        constexpr int R = decltype(r)::value;
        constexpr bool BF = decltype(bf)::value;
        if (int rc = place_bc<T>(a, pl, bc, stream, "vsv_ssm_scan")) return rc;
        if (pl.S > 1) {
            hipLaunchKernelGGL((ssm_ends_kernel<T, R, BF>), dim3((unsigned)(waves * (pl.S - 1))), dim3(64), 0, (hipStream_t)stream, *a, pl, E, sd);
            if (int rc = op_launch_check("ssm_ends_kernel")) return rc;
        }
        hipLaunchKernelGGL((ssm_scan_kernel<T, R, BF>), dim3((unsigned)(waves * pl.S)), dim3(64), 0, (hipStream_t)stream, *a, pl, E, sd);
        return op_launch_check("ssm_scan_kernel");
    });
}

namespace {
size_t part_bc_floats(const vsv_ssm_desc* a) { return (size_t)ssm_blocks(a) * a->B * a->T * a->G * 2 * padded_states(a->N); }
}  // namespace

extern "C" size_t vsv_ssm_scan_backward_ws_bytes(const vsv_ssm_desc* a) {
    if (check_ssm(a, "vsv_ssm_scan_backward_ws_bytes")) return 0;
    const ScanPlan pl = scan_plan(a);
    return (round4(bc_floats(a)) + round4(ends_floats(a, pl)) + round4(part_bc_floats(a)) +
            (size_t)a->B * pl.S * (padded_states(a->N) + 2) * a->D) * sizeof(float);
}

extern "C" int vsv_ssm_scan_backward(const vsv_ssm_desc* a, const vsv_ssm_grads* g, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_ssm(a, "vsv_ssm_scan_backward")) return rc;
    if (!g || (a->B > 0 && a->T > 0 && (!a->saved || !g->dy || !g->dx || !g->ddt || !g->db || !g->dc || (a->gate && !g->dgate)))) {
        set_error("vsv_ssm_scan_backward: null pointer"); return -1;
    }
    if (ws_bytes < vsv_ssm_scan_backward_ws_bytes(a) || (a->B > 0 && (!ws || !aligned(ws, 16)))) {
        set_error("vsv_ssm_scan_backward: workspace too small or not on 16 bytes"); return -1;
    }
    if (a->saved && !aligned(a->saved, 16)) { set_error("vsv_ssm_scan_backward: saved must be on 16 bytes"); return -1; }
    ScanPlan pl = scan_plan(a);
    const int R0 = padded_states(a->N);
    const long nb = ssm_blocks(a), waves = a->B * a->G * nb, rows = a->B * a->T * a->G;
    if (waves * pl.S > kMaxBlocks || (rows * 2 * R0 + 255) / 256 > kMaxBlocks) { set_error("vsv_ssm_scan_backward: too many elements for one call"); return -2; }
    float *bc = (float*)ws, *E = bc + round4(bc_floats(a)), *sd = E + (size_t)a->B * pl.S * R0 * a->D;
    float *pbc = E + round4(ends_floats(a, pl)), *pp = pbc + round4(part_bc_floats(a));
    if (a->B > 0) {
        const int rc = by_scan(a, "vsv_ssm_scan_backward", [&](auto t, auto r, auto bf) {
            using T = decltype(t);
            constexpr int R = decltype(r)::value;
            constexpr bool BF = decltype(bf)::value;
            if (int rc = place_bc<T>(a, pl, bc, stream, "vsv_ssm_scan_backward")) return rc;
            if (pl.S > 1) {
                hipLaunchKernelGGL((ssm_bwd_ends_kernel<T, R, BF>), dim3((unsigned)(waves * (pl.S - 1))), dim3(64), 0, (hipStream_t)stream, *a, *g, pl, E, sd);
                if (int rc = op_launch_check("ssm_bwd_ends_kernel")) return rc;
            }
            hipLaunchKernelGGL((ssm_bwd_kernel<T, R, BF>), dim3((unsigned)(waves * pl.S)), dim3(64), 0, (hipStream_t)stream, *a, *g, pl, E, sd, pbc, pp);
            if (int rc = op_launch_check("ssm_bwd_kernel")) return rc;
            if (rows == 0) return 0;
            hipLaunchKernelGGL(sum_bc_kernel<T>, dim3((unsigned)((rows * 2 * R + 255) / 256)), dim3(256), 0, (hipStream_t)stream, pbc, nb, rows, R, a->N, (T*)g->db, (T*)g->dc);
            return op_launch_check("sum_bc_kernel");
        });
        if (rc) return rc;
    }
    hipLaunchKernelGGL(sum_params_kernel, dim3((unsigned)(((R0 + 2) * a->D + 63) / 64)), dim3(256), 0, (hipStream_t)stream, pp, a->B * pl.S, a->D, R0, a->N, g->da, g->dskip, g->ddt_bias);
    return op_launch_check("sum_params_kernel");
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
