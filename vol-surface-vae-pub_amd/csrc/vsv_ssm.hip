// Selective state space memory: the short causal convolution, the scan, their backward passes and their single-token
// forms.  Rows are (sequence, time step), features are contiguous; states, statistics and parameter gradients are
// float32 whatever the sequences' type.
#include <cfloat>
#include <type_traits>

#include "vsv_ops.h"

namespace vsv {
namespace {

__device__ inline long seq_len(const int* lengths, long b, long T) {
    if (!lengths) return T;
    const long n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}

// ---- short causal convolution ------------------------------------------------------------------------------------
// One output from the window, tap by tap and each operation rounded by itself: a prompt and the tokens behind it come out
// bit for bit the same, whichever kernel computes them, and so does any evaluation that takes the formula at its word -- what
// is rounded to 16 bits here feeds a recurrent state.  exp(-s) is 2^t with what t = -s log2 e is rounded by put behind it; the
// quotient 1 / (1 + e) is the reciprocal with one Newton step (a full division costs ten operations more).
template <int K>
__device__ inline float conv_pre(const float (&w)[K], const float (&x)[K], float bias) {
#pragma clang fp contract(off)
    float s = w[0] * x[0];
#pragma unroll
    for (int k = 1; k < K; ++k) s = s + w[k] * x[k];
    return s + bias;
}
__device__ inline float conv_silu(float s) {
    constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f, kLn2 = 0.693147182f;       // log2 e, what it is rounded by, 1 / log2 e
    const float x = __builtin_amdgcn_fmed3f(-s, -100.0f, 88.0f), t = x * kHi;
    const float e = exp2_fast(t) * __builtin_fmaf(__builtin_fmaf(x, kLo, __builtin_fmaf(x, kHi, -t)), kLn2, 1.0f);
    const float y = 1.0f + e, r = __builtin_amdgcn_rcpf(y);                // (e^88 is the largest that leaves it finite)
    return s * __builtin_fmaf(__builtin_fmaf(-y, r, 1.0f), r, r);
}

// pre[t,d] = bias[d] + sum_k w[d,k] xs[t-K+1+k, d],  y = silu(pre) or pre; xs is x, continued into state_in before t = 0.
// One read of x and one write of y (2K flops an element): bound by memory (8x2048x4096 bf16: 57 to 61 us, 4.4 to 4.7 TB/s).  A thread owns VEC
// neighbouring channels and a chunk of time, so the window stays in registers and only K-1 rows per chunk are read twice; it
// works on kRows rows at a time, with the next ones under way.
template <typename T, int K, int VEC, int kRows> struct ConvRows {
    const T* x;                      // the sequence's row 0, at this thread's channels
    const float* st;                 // state_in's, or null
    long ts, D, len;
    Pack<T, VEC> raw[kRows];
    __device__ inline ConvRows(const vsv_short_conv_desc& a, long b, long d0)
        : x((const T*)a.x + b * a.x_bs + d0), st(a.state_in ? a.state_in + b * (K - 1) * a.D + d0 : nullptr), ts(a.x_ts), D(a.D),
          len(seq_len(a.lengths, b, a.T)) {}
    __device__ inline void row(long t, float (&out)[VEC]) const {          // xs[t] for any t < len, zeros from there on
        if (t >= 0 && t < len) { load_vec<T, VEC>(x + t * ts, out); return; }
#pragma unroll
        for (int v = 0; v < VEC; ++v) out[v] = t < 0 && st ? st[(t + K - 1) * D + v] : 0.0f;
    }
    __device__ inline void fetch(const T* at) {                            // kRows rows from here on
#pragma unroll
        for (int u = 0; u < kRows; ++u) raw[u] = *reinterpret_cast<const Pack<T, VEC>*>(at + u * ts);
    }
    __device__ inline void take(int u, float (&out)[VEC]) const {
#pragma unroll
        for (int v = 0; v < VEC; ++v) out[v] = to_f(raw[u].v[v]);
    }
};

template <typename T, int K, int VEC, int kRows>
__global__ void __launch_bounds__(256) short_conv_kernel(const vsv_short_conv_desc a, long chunk, long n_chunk, long n_vec) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.B * n_chunk * n_vec) return;
    const long dv = id % n_vec, bc = id / n_vec, ch = bc % n_chunk, b = bc / n_chunk;
    const long d0 = dv * VEC, t0 = ch * chunk, t1 = t0 + chunk < a.T ? t0 + chunk : a.T;
    T* y = (T*)a.y + b * a.T * a.D + d0;
    ConvRows<T, K, VEC, kRows> in(a, b, d0);
    float w[VEC][K], bias[VEC], xs[K - 1 + kRows][VEC];
    const long lim = t1 < in.len ? t1 : in.len;                           // rows from here on to t1 are padding
    const T* px = in.x + t0 * in.ts;
    if (t0 + kRows <= lim) in.fetch(px);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) in.row(t0 - K + 1 + k, xs[k]);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        bias[v] = a.bias ? a.bias[d0 + v] : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[v][k] = a.w[(d0 + v) * K + k];
    }
    auto put = [&](int u, T* to) {
        float out[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float win[K];
#pragma unroll
            for (int k = 0; k < K; ++k) win[k] = xs[u + k][v];
            out[v] = conv_pre<K>(w[v], win, bias[v]);
        }
        if (a.silu) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) out[v] = conv_silu(out[v]);
        }
        store_vec<T, VEC>(to, out);
    };
    long t = t0;
    y += t0 * a.D;
    for (; t + kRows <= lim; t += kRows) {
#pragma unroll
        for (int u = 0; u < kRows; ++u) in.take(u, xs[K - 1 + u]);
        if (t + 2 * kRows <= lim) { px += kRows * in.ts; in.fetch(px); }
#pragma unroll
        for (int u = 0; u < kRows; ++u, y += a.D) put(u, y);
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) xs[k][v] = xs[k + kRows][v];
    }
    for (; t < lim; ++t, y += a.D) {
        in.row(t, xs[K - 1]);
        put(0, y);
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) xs[k][v] = xs[k + 1][v];
    }
    const float zeros[VEC] = {};
    for (; t < t1; ++t, y += a.D) store_vec<T, VEC>(y, zeros);
    if (a.state_out && ch == 0) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            float r[VEC];
            in.row(in.len - (K - 1) + j, r);
#pragma unroll
            for (int v = 0; v < VEC; ++v) a.state_out[(b * (K - 1) + j) * a.D + d0 + v] = r[v];
        }
    }
}

// ds = dy act'(pre) (pre computed again from x), dx[t] = sum_k w[k] ds[t+K-1-k], dw[k] = sum_t ds[t] xs[t-K+1+k],
// dbias = sum_t ds.  The same chunks; a chunk reads K-1 rows beyond each end, its sums over time go to `part`
// (chunk, K + 1, D) and are joined in a fixed order by sum_conv_parts_kernel.  8x2048x4096 bf16: 90 us, 4.5 TB/s; 16x8192x515, a
// channel a thread in accesses of two bytes: 232 us, 16x8192x516: 145.
template <typename T, int K, int VEC, int kRows>
__global__ void __launch_bounds__(256) short_conv_bwd_kernel(const vsv_short_conv_desc a, const vsv_short_conv_grads g, long chunk, long n_chunk,
                                                             long n_vec, float* __restrict__ part) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.B * n_chunk * n_vec) return;
    const long dv = id % n_vec, bc = id / n_vec, ch = bc % n_chunk, b = bc / n_chunk;
    const long d0 = dv * VEC, t0 = ch * chunk, t1 = t0 + chunk < a.T ? t0 + chunk : a.T;
    const T* dy = (const T*)g.dy + b * g.dy_bs + d0;
    T* dx = (T*)g.dx + b * a.T * a.D + d0;
    const float* dso = g.d_state_out ? g.d_state_out + b * (K - 1) * a.D + d0 : nullptr;
    ConvRows<T, K, VEC, kRows> in(a, b, d0);
    Pack<T, VEC> dyr[kRows];
    float w[K][VEC], bias[VEC], xs[K - 1 + kRows][VEC], ds[K - 1 + kRows][VEC], dw[K][VEC], db[VEC];
    const long lim = t1 < in.len ? t1 : in.len;
    const T *px = in.x + t0 * in.ts, *pdy = dy + t0 * g.dy_ts;
    auto fetch = [&] {
        in.fetch(px);
#pragma unroll
        for (int u = 0; u < kRows; ++u) dyr[u] = *reinterpret_cast<const Pack<T, VEC>*>(pdy + u * g.dy_ts);
    };
    if (t0 + kRows <= lim) fetch();
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        in.row(t0 - K + 1 + k, xs[k]);
#pragma unroll
        for (int v = 0; v < VEC; ++v) ds[k][v] = 0.0f;
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        bias[v] = a.bias ? a.bias[d0 + v] : 0.0f;
        db[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) { w[k][v] = a.w[(d0 + v) * K + k]; dw[k][v] = 0.0f; }
    }
    auto slope = [&](int u, int v, float d) {                             // dy act'(pre) at the window that ends in xs[K - 1 + u]
        if (!a.silu) return d;
        float s = bias[v];
#pragma unroll
        for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][v], xs[u + k][v], s);
        const float sg = sigmoid_f(s);
        return d * sg * __builtin_fmaf(s, 1.0f - sg, 1.0f);
    };
    auto weigh = [&](int u) {                                             // a row's share of dw and db
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float d = ds[K - 1 + u][v];
            db[v] += d;
#pragma unroll
            for (int k = 0; k < K; ++k) dw[k][v] = __builtin_fmaf(d, xs[u + k][v], dw[k][v]);
        }
    };
    auto back = [&](int u, float (&o)[VEC]) {                             // dx of the row K - 1 in front: ds[to + K-1-k] is ds[u + K-1-k] here
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            o[v] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) o[v] = __builtin_fmaf(w[k][v], ds[u + K - 1 - k][v], o[v]);
        }
    };
    auto shift = [&](int rows) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) { xs[k][v] = xs[k + rows][v]; ds[k][v] = ds[k + rows][v]; }
    };
    const long lo = ch == 0 ? -(K - 1) : t0, end = t1 + K - 1;            // (chunk 0 also returns the state's gradient)
    auto give = [&](long to, const float (&o)[VEC]) {
        if (to >= 0) store_vec<T, VEC>(dx + to * a.D, o);
        else if (g.d_state_in) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) g.d_state_in[(b * (K - 1) + to + K - 1) * a.D + d0 + v] = o[v];
        }
    };
    long t = t0;
    for (; t + kRows <= lim; t += kRows) {                                // rows of the chunk, none of them padding
        float dyv[kRows][VEC];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            in.take(u, xs[K - 1 + u]);
#pragma unroll
            for (int v = 0; v < VEC; ++v) dyv[u][v] = to_f(dyr[u].v[v]);
        }
        if (t + 2 * kRows <= lim) { px += kRows * in.ts; pdy += kRows * g.dy_ts; fetch(); }
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) ds[K - 1 + u][v] = slope(u, v, dyv[u][v]);
            weigh(u);
            float o[VEC];
            back(u, o);
            const long to = t + u - (K - 1);
            if (to >= lo) give(to, o);
        }
        shift(kRows);
    }
    for (; t < end; ++t) {                                                // what is left of it, and the K - 1 rows behind it
        in.row(t, xs[K - 1]);
        float dyv[VEC] = {}, o[VEC];
        if (t < in.len) load_vec<T, VEC>(dy + t * g.dy_ts, dyv);
#pragma unroll
        for (int v = 0; v < VEC; ++v) ds[K - 1][v] = t < in.len ? slope(0, v, dyv[v]) : 0.0f;
        if (t < lim) weigh(0);
        back(0, o);
        const long to = t - (K - 1), jj = to - (in.len - (K - 1));        // (the row of state_out that xs[to] is, if any)
        if (dso && jj >= 0 && jj < K - 1) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] += dso[jj * a.D + v];
        }
        if (to >= lo && to < t1) give(to, o);
        shift(1);
    }
    float* p = part + (b * n_chunk + ch) * (K + 1) * a.D + d0;
#pragma unroll
    for (int k = 0; k < K; ++k) store_vec<float, VEC>(p + k * a.D, dw[k]);
    store_vec<float, VEC>(p + (long)K * a.D, db);
}

// out_j = sum over rows of part (rows, M); element m = k * D + d goes to dw[d * K + k] or, k == K, to dbias[d].  A workgroup has 64
// columns and all rows: 5 us where the channels are many (8x2048x4096), but 87 beside the pass's own 88 for 8192 rows of 64 channels
// (64x16384x64), bound by the latency of a walk eight loads deep.
__global__ void __launch_bounds__(256) sum_conv_parts_kernel(const float* __restrict__ part, long rows, long D, int K,
                                                             float* __restrict__ dw, float* __restrict__ dbias) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long M = (K + 1) * D, m = (long)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (m < M) {
#pragma unroll 8
        for (long r = wave; r < rows; r += 4) s += part[r * M + m];
    }
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
    const float s = conv_pre<K>(wv, win, bias ? bias[d] : 0.0f);
    y[b * D + d] = from_f<T>(silu ? conv_silu(s) : s);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) state[(b * (K - 1) + k) * D + d] = win[k + 1];
}

// ---- selective scan ----------------------------------------------------------------------------------------------
// delta = softplus(dt + dt_bias),  h_t = exp(delta a) h_{t-1} + delta x b_t,  y = (c_t . h_t + skip x) silu(gate).
// The decay belongs to (channel, state), so there is no matrix form: per state and step one exponential and four float32
// operations, 24 cycles of a SIMD per 64 channels, against 8 bytes of traffic per channel and step in 16 bits.  Bound by
// the vector units: 1x16384x2048 bf16 takes 268 us in all, of which the issue of its vector instructions is 227; 256x512x1024, which
// is not split, 557 us (375 at 24 cycles a state).
//   A lane owns a channel and its N states (padded to R) in registers (or four of them), a wave 64 channels of one group (or
// 256 / R), which share b_t and c_t.  x, dt, gate, b and c of the next kTile steps are loaded while the present ones are
// computed; the activations are taken for a tile at a time.
//   A wave runs along time alone, so where sequences and channels make fewer waves than the chip has SIMDs the time axis is
// split (scan_plan).  A first pass gives every segment's state from zero and its sum of delta; the state in front of a
// segment then follows from exp(a sum delta), one step per earlier segment: at the start of the second pass or, of many
// segments, between the two.
constexpr int kTile = 8;             // steps per tile; training keeps the state before every tile

struct ScanPlan {
    long seg;                        // steps per segment, a multiple of kTile
    int S;                           // segments
    int P;                           // lanes that share a channel's states (forward)
    bool joined;                     // the states in front of the segments come from ssm_join_kernel
};

struct ScanPos {
    long b, g, base, t0, t1, tz;     // sequence, group, first channel; the segment's steps [t0, t1), padding [t1, tz)
    int s;
    unsigned lane;                   // channel base + lane
    int part;                        // which R / P of its states this lane owns
    bool live;                       // a channel of its own
};

__device__ inline long seq_len_s(const int* lengths, long b, long T) {
    if (!lengths) return T;
    const long n = ((const __attribute__((address_space(4))) int*)(uintptr_t)lengths)[b];
    return n < 0 ? 0 : n > T ? T : n;
}

template <int P = 1> __device__ inline ScanPos scan_pos(const vsv_ssm_desc& a, const ScanPlan& pl, unsigned blk, int s0) {
    constexpr unsigned kCh = 64 / P;
    const unsigned Dg = (unsigned)(a.D / a.G), cb = (Dg + kCh - 1) / kCh, ch = threadIdx.x % kCh;
    const unsigned w = (unsigned)(a.B * a.G) * cb;
    ScanPos p;
    p.s = (int)(blk / w) + s0;
    blk %= w;
    const unsigned c = blk % cb, bg = blk / cb;
    p.g = bg % (unsigned)a.G;
    p.b = bg / (unsigned)a.G;
    p.base = p.g * Dg + c * kCh;
    const unsigned left = Dg - c * kCh;
    p.part = threadIdx.x / kCh;
    p.live = ch < left;
    p.lane = p.live ? ch : left - 1;
    const long len = seq_len_s(a.lengths, p.b, a.T);
    p.t0 = p.s * pl.seg;
    p.tz = p.t0 + pl.seg < a.T ? p.t0 + pl.seg : a.T;
    p.t1 = p.tz < len ? p.tz : len;
    return p;
}

// An empty statement that a value passes through: what is computed from it stays behind it, in its step.  (Without it the
// steps of a tile are computed side by side, and their states do not fit the registers.)
__device__ inline void pin(float& v) { asm volatile("" : "+v"(v)); }
__device__ inline void order() { __builtin_amdgcn_sched_barrier(0); }

// Orders what the lanes of a wave store to shared memory and load from it (a workgroup is one wave; this is no instruction).
__device__ inline void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// b and c of a tile: eight lanes to a step, four of them b's states and four c's, R / 4 each.  They are loaded a tile ahead,
// whatever their strides, and laid down in the wave's own shared memory as float32, zeros behind the N states; a step then
// reads its rows as broadcasts.  (Read through the scalar cache, with the next step's rows under way during the present
// step, 64x60x100 in float32 took 32 us for 26: the scalar loads miss to L2, and only the latest can be waited for.)
template <typename T, int R> struct BcTile {
    static constexpr int V = R / 4;
    const T* at;                     // this lane's first state in the tile's first row of its own
    long ts;
    int row, n0, to;
    bool on;
    T raw[V];
    __device__ inline BcTile(const vsv_ssm_desc& a, const ScanPos& p, long t, bool use_b, bool use_c) {
        const int l = threadIdx.x, c = (l >> 2) & 1;
        row = l >> 3;
        n0 = (l & 3) * V;
        to = row * 2 * R + c * R + n0;
        on = c ? use_c : use_b;
        ts = c ? a.c_ts : a.b_ts;
        at = (const T*)(c ? a.c : a.b) + p.b * (c ? a.c_bs : a.b_bs) + p.g * (c ? a.c_gs : a.b_gs) + (t + row) * ts + n0;
    }
    __device__ inline void fetch(int N, int left) {                       // rows behind the first `left` repeat the last
        if (!on) return;
        const T* q = at;
        if (left < kTile && row >= left) q -= (row - left + 1) * ts;
#pragma unroll
        for (int k = 0; k < V; ++k) raw[k] = n0 + k < N ? q[k] : from_f<T>(0.0f);
    }
    __device__ inline void move(int tiles) { at += (long)tiles * kTile * ts; }
    __device__ inline void lay(float* lds) const {
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = to_f(raw[k]);
        wave_fence();
        if (on) store_vec<float, V>(lds + to, v);
        wave_fence();
    }
};
// H states of a row, the same for every lane
template <int H> __device__ inline void bc_row(const float* lds, float (&v)[H]) {
#pragma unroll
    for (int k = 0; k < H / 4; ++k) {
        float q[4];
        load_vec<float, 4>(lds + 4 * k, q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * k + j] = q[j];
    }
}

// One channel per lane of kTile rows from `row` on, `step` bytes apart (rows behind the first `left` repeat the last):
// buffer loads, whose per-row address is one scalar offset.
template <typename T> __device__ inline T buffer_get(__amdgpu_buffer_rsrc_t r, unsigned voff, int soff) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, soff, 0));
    else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(r, (int)voff, soff, 0));
}
template <typename T>
__device__ inline void load_tile(const T* row, int step, unsigned lane, int left, T (&out)[kTile]) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(row), 0, -1, 0x00020000);
#pragma unroll
    for (int i = 0; i < kTile; ++i) out[i] = buffer_get<T>(r, lane * (unsigned)sizeof(T), (i < left ? i : left - 1) * step);
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
// (a dead lane's offset lies behind the buffer's end, where stores are dropped)
template <typename T> __device__ inline void tile_store(T* row, long D, const ScanPos& p, int left, const float (&v)[kTile]) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc(row, 0, 0x7fffffff, 0x00020000);
    const int voff = p.live ? (int)(p.lane * (unsigned)sizeof(T)) : (int)0xfffffff0;
    const int step = (int)(D * (long)sizeof(T));
#pragma unroll
    for (int i = 0; i < kTile; ++i) {
        if (left < kTile && i >= left) break;
        const T o = from_f<T>(v[i]);
        if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, o), r, voff, i * step, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, o), r, voff, i * step, 0);
    }
}

// decay_n = exp(delta a_n), all of them before the first is used: an exponential's result is late
template <int R> __device__ inline void decays(float de, const float* A2, float (&e)[R]) {
#pragma unroll
    for (int n = 0; n < R; ++n) e[n] = de * A2[n];
#pragma unroll
    for (int n = 0; n < R; ++n) e[n] = exp2_fast(e[n]);
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

// a log2 e.  A state that is forgotten at once (a = -inf, or below what float32 holds of the product) stays finite here: padding's
// delta of 0 must leave it as it is, and 0 times infinity would not.
__device__ inline float decay_exponent(float a) {
    const float x = a * kLog2e;
    return x < -FLT_MAX ? -FLT_MAX : x;
}
template <int R> __device__ inline void load_decay(const vsv_ssm_desc& a, long d, float (&A2)[R], int n0 = 0) {
#pragma unroll
    for (int n = 0; n < R; ++n) A2[n] = n0 + n < a.N ? decay_exponent(a.a[d * a.N + n0 + n]) : 0.0f;
}

// Between the P lanes of a channel, 64 / P apart, of which lane `part` owns steps part kTile / P + j of a tile: values of the
// own steps to all steps' in every lane, and every lane's shares of all steps to the own steps' sums.
__device__ inline void swap32(float a, float b, float& r0, float& r1) {   // (a.lo, b.lo), (a.hi, b.hi) of the wave's halves
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned x = r[0], y = r[1];
    r0 = __builtin_bit_cast(float, x);
    r1 = __builtin_bit_cast(float, y);
}
__device__ inline void swap16(float a, float b, float& r0, float& r1) {   // the same within each half
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned x = r[0], y = r[1];
    r0 = __builtin_bit_cast(float, x);
    r1 = __builtin_bit_cast(float, y);
}
template <int P> __device__ inline void to_all(const float (&own)[kTile / P], float (&all)[kTile]) {
    static_assert(P == 2 || P == 4, "");
    float h[kTile / 2];
    if constexpr (P == 4) {
#pragma unroll
        for (int j = 0; j < kTile / 4; ++j) swap16(own[j], own[j], h[j], h[j + kTile / 4]);
    } else {
#pragma unroll
        for (int j = 0; j < kTile / 2; ++j) h[j] = own[j];
    }
#pragma unroll
    for (int j = 0; j < kTile / 2; ++j) swap32(h[j], h[j], all[j], all[j + kTile / 2]);
}
template <int P> __device__ inline void sums_to_own(const float (&all)[kTile], float (&own)[kTile / P]) {
    float h[kTile / 2], u, v;
#pragma unroll
    for (int j = 0; j < kTile / 2; ++j) { swap32(all[j], all[j + kTile / 2], u, v); h[j] = u + v; }
    if constexpr (P == 4) {
#pragma unroll
        for (int j = 0; j < kTile / 4; ++j) { swap16(h[j], h[j + kTile / 4], u, v); own[j] = u + v; }
    } else {
#pragma unroll
        for (int j = 0; j < kTile / 2; ++j) own[j] = h[j];
    }
}

// 2^x v + e where 2^x may leave float32 (states that grow): a v of 0 stays 0, any other takes the factor in two halves.
__device__ inline float carry_past(float x, float v, float e) {
    const float half = exp2_fast(0.5f * x);
    return v == 0.0f ? e : __builtin_fmaf(v * half, half, e);
}

// v = exp(a sum delta) v + E over the segments from, from + step, .. up to (not including) to, from v = first(); the loads of
// kAhead of them are under way at a time.  Should a factor of any lane leave float32, all of it once more, one segment at a time.  (A
// branch in the loop itself costs ssm_scan_kernel a third of its waves, in registers; one that the lanes take apart costs ssm_bwd_kernel
// 20 us of 270, in scalar registers that leave its loop for lanes of vector registers.)
template <int R, typename F>
__device__ inline void fold_segments(const float* E, const float* sd, long row_floats, long D, long d, long row0, int from, int to, int step,
                                     const float (&A2)[R], float (&v)[R], int N, F&& first) {
    constexpr int kAhead = 4;
    const int n = (to - from) * step;
    float top = 0.0f;
    first(v, N);
    for (int i = 0; i < n; i += kAhead) {
        float e[kAhead][R], s[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const long k = row0 + from + (i + u < n ? i + u : n - 1) * step;
            load_states<R>(E + k * row_floats, D, d, e[u]);
            s[u] = sd[k * D + d];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            pin(s[u]);
#pragma unroll
            for (int m = 0; m < R; ++m) pin(e[u][m]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i + u >= n) break;
            float w[R];
            decays<R>(s[u], A2, w);
#pragma unroll
            for (int m = 0; m < R; ++m) {
                v[m] = __builtin_fmaf(w[m], v[m], e[u][m]);
                top = __builtin_fmaxf(top, w[m]);
            }
        }
    }
    if (!__any(top > FLT_MAX)) return;
    int again = N;
    asm volatile("" : "+s"(again));                                       // (or the first time's n < N are kept until here)
    first(v, again);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const long k = row0 + from + i * step;
        float e[R], w[R];
        load_states<R>(E + k * row_floats, D, d, e);
        const float s = sd[k * D + d];
        decays<R>(s, A2, w);
#pragma unroll
        for (int m = 0; m < R; ++m) v[m] = w[m] > FLT_MAX ? carry_past(s * A2[m], v[m], e[m]) : __builtin_fmaf(w[m], v[m], e[m]);
    }
}

// The same for many segments, in a launch between the passes: E becomes the state in front of every segment (behind it,
// backwards), so that a segment does not walk over all the others'.  A lane has one state of a channel.
template <int R>
__global__ void __launch_bounds__(64) ssm_join_kernel(const float* __restrict__ a, const float* __restrict__ init, int N, long D, long rows,
                                                      int S, bool back, float* __restrict__ E, const float* __restrict__ sd) {
    constexpr int kAhead = 16;
    const long id = (long)blockIdx.x * 64 + threadIdx.x;
    if (id >= rows * R * D) return;
    const long b = id / (R * D), at = id - b * R * D, k = at / (4 * D), d = (at - k * 4 * D) >> 2;
    const int n = (int)(k * 4 + (at & 3));
    const float A2 = n < N ? decay_exponent(a[d * N + n]) : 0.0f;
    float v = n < N && init ? init[(b * D + d) * N + n] : 0.0f;
    for (int i = 0; i < S; i += kAhead) {
        float e[kAhead], s[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = i + u < S - 1 ? i + u : S - 2;
            const long row = b * S + (back ? S - 1 - j : j);
            e[u] = E[row * R * D + at];
            s[u] = sd[row * D + d];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) { pin(e[u]); pin(s[u]); }         // (all of them under way, none loaded behind the break)
        float w[kAhead], top = 0.0f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            w[u] = exp2_fast(s[u] * A2);
            top = __builtin_fmaxf(top, w[u]);
        }
        auto take = [&](auto past) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (i + u >= S) break;
                E[(b * S + (back ? S - 1 - i - u : i + u)) * R * D + at] = v;
                v = past.value && w[u] > FLT_MAX ? carry_past(s[u] * A2, v, e[u]) : __builtin_fmaf(w[u], v, e[u]);
            }
        };
        if (__any(top > FLT_MAX)) take(std::true_type{});
        else take(std::false_type{});
    }
}

// First pass of a split scan: a segment's last state from zero, and its sum of delta.
template <typename T, int R>
__global__ void __launch_bounds__(64) ssm_ends_kernel(const vsv_ssm_desc a, const ScanPlan pl, float* __restrict__ E, float* __restrict__ sd) {
    __shared__ alignas(16) float lds[2][kTile * 2 * R];
    const ScanPos p = scan_pos(a, pl, blockIdx.x, 0);
    const long D = a.D, d = p.base + p.lane;
    float A2[R], h[R] = {}, sum = 0.0f;
    load_decay<R>(a, d, A2);
    const float dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    const T *x = (const T*)a.x + p.b * a.x_bs + p.base + p.t0 * a.x_ts, *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + p.t0 * a.dt_ts;
    BcTile<T, R> bc(a, p, p.t0, true, false);
    T xr[kTile], dr[kTile];
    auto fetch = [&](int left) {
        bc.fetch(a.N, left);
        load_tile(x, (int)(a.x_ts * (long)sizeof(T)), p.lane, left, xr);
        load_tile(dt, (int)(a.dt_ts * (long)sizeof(T)), p.lane, left, dr);
    };
    if (p.t0 < p.t1) fetch(tile_left(p, p.t0));
    int buf = 0;
    for (long t = p.t0; t < p.t1; t += kTile, buf ^= 1) {
        const int left = tile_left(p, t);
        float xv[kTile], raw[kTile], de[kTile];
        bc.lay(lds[buf]);
        tile_values(xr, left, xv);
        tile_steps(dr, dtb, a.softplus, left, raw, de);
        if (t + kTile < p.t1) {
            x += kTile * a.x_ts; dt += kTile * a.dt_ts; bc.move(1);
            fetch(tile_left(p, t + kTile));
        }
        order();
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            float b[R], e[R];
            bc_row<R>(lds[buf] + i * 2 * R, b);
            const float dx = de[i] * xv[i];
            decays<R>(de[i], A2, e);
            sum += de[i];
            order();
#pragma unroll
            for (int n = 0; n < R; ++n) h[n] = __builtin_fmaf(e[n], h[n], dx * b[n]);
            order();
        }
    }
    if (!p.live) return;
    store_states<R>(E + (p.b * pl.S + p.s) * R * D, D, d, h);
    sd[(p.b * pl.S + p.s) * D + d] = sum;
}

// The outputs, from the state in front of the segment on.
template <typename T, int R>
__global__ void __launch_bounds__(64) ssm_scan_kernel(const vsv_ssm_desc a, const ScanPlan pl, const float* __restrict__ E,
                                                      const float* __restrict__ sd) {
    __shared__ alignas(16) float lds[2][kTile * 2 * R];
    const ScanPos p = scan_pos(a, pl, blockIdx.x, 0);
    const long D = a.D, d = p.base + p.lane;
    const int N = a.N;
    T* y = (T*)a.y + p.b * a.T * D + p.base;
    const T *x = (const T*)a.x + p.b * a.x_bs + p.base + p.t0 * a.x_ts, *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + p.t0 * a.dt_ts;
    const T* gate = a.gate ? (const T*)a.gate + p.b * a.gate_bs + p.base + p.t0 * a.gate_ts : nullptr;
    BcTile<T, R> bc(a, p, p.t0, true, true);
    T xr[kTile], dr[kTile], gr[kTile];
    auto fetch = [&](int left) {
        bc.fetch(N, left);
        load_tile(x, (int)(a.x_ts * (long)sizeof(T)), p.lane, left, xr);
        load_tile(dt, (int)(a.dt_ts * (long)sizeof(T)), p.lane, left, dr);
        if (gate) load_tile(gate, (int)(a.gate_ts * (long)sizeof(T)), p.lane, left, gr);
    };
    if (p.t0 < p.t1) fetch(tile_left(p, p.t0));
    float A2[R], h[R];
    load_decay<R>(a, d, A2);
    auto first = [&](float (&v)[R], int N) {
#pragma unroll
        for (int n = 0; n < R; ++n) v[n] = n < N && a.state_in ? a.state_in[(p.b * D + d) * N + n] : 0.0f;
    };
    if (pl.joined) load_states<R>(E + (p.b * pl.S + p.s) * R * D, D, d, h);
    else fold_segments<R>(E, sd, R * D, D, d, p.b * pl.S, 0, p.s, 1, A2, h, N, first);
    const float skip = a.skip ? a.skip[d] : 0.0f, dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    float* saved = a.saved ? a.saved + (p.b * ((a.T + kTile - 1) / kTile) + p.t0 / kTile) * R * D : nullptr;
    int buf = 0;
    for (long t = p.t0; t < p.t1; t += kTile, buf ^= 1) {
        const int left = tile_left(p, t);
        float xv[kTile], raw[kTile], de[kTile], gv[kTile], yv[kTile];
        bc.lay(lds[buf]);
        tile_values(xr, left, xv);
        tile_steps(dr, dtb, a.softplus, left, raw, de);
        if (gate) {
            tile_values(gr, left, gv);
#pragma unroll
            for (int i = 0; i < kTile; ++i) gv[i] *= sigmoid_f(gv[i]);
        }
        if (t + kTile < p.t1) {
            x += kTile * a.x_ts; dt += kTile * a.dt_ts; gate += gate ? kTile * a.gate_ts : 0; bc.move(1);
            fetch(tile_left(p, t + kTile));
        }
        if (saved) {
            if (p.live) store_states<R>(saved, D, d, h);
            saved += R * D;
        }
        order();
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            float b[R], c[R], e[R], acc[2] = {skip * xv[i], 0.0f};
            bc_row<R>(lds[buf] + i * 2 * R, b);
            bc_row<R>(lds[buf] + i * 2 * R + R, c);
            const float dx = de[i] * xv[i];
            decays<R>(de[i], A2, e);
            order();
#pragma unroll
            for (int n = 0; n < R; ++n) {
                h[n] = __builtin_fmaf(e[n], h[n], dx * b[n]);
                acc[n & 1] = __builtin_fmaf(c[n], h[n], acc[n & 1]);
            }
            yv[i] = acc[0] + acc[1];
            order();
        }
        if (gate) {
#pragma unroll
            for (int i = 0; i < kTile; ++i) yv[i] *= gv[i];
        }
        tile_store(y + t * D, D, p, left, yv);
    }
    if (p.live)
        for (long t = p.t0 > p.t1 ? p.t0 : p.t1; t < p.tz; ++t) (y + t * D)[p.lane] = from_f<T>(0.0f);
    if (a.state_out && p.live && p.s == pl.S - 1)
#pragma unroll
        for (int n = 0; n < R; ++n)
            if (n < N) a.state_out[(p.b * D + d) * N + n] = h[n];
}

// Both passes where waves are few: P = R / 4 lanes share a channel, four states each.  A wave is alone on its SIMD and every
// instruction counts, so a tile's steps are shared too: a lane loads, activates, gates and stores kTile / P of them.  ENDS: the
// first pass.
template <typename T, int R, int P, bool ENDS>
__global__ void __launch_bounds__(64) ssm_shared_kernel(const vsv_ssm_desc a, const ScanPlan pl, float* __restrict__ E, float* __restrict__ sd) {
    __shared__ alignas(16) float lds[2][kTile * 2 * R];
    constexpr int L = R / P, O = kTile / P;
    constexpr unsigned kSize = sizeof(T);
    const ScanPos p = scan_pos<P>(a, pl, blockIdx.x, 0);
    const long D = a.D, d = p.base + p.lane;
    const int N = a.N, n0 = p.part * L, own = p.part * O;                 // the first of this lane's states and steps
    const T *x = (const T*)a.x + p.b * a.x_bs + p.base + p.t0 * a.x_ts, *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + p.t0 * a.dt_ts;
    const T* gate = !ENDS && a.gate ? (const T*)a.gate + p.b * a.gate_bs + p.base + p.t0 * a.gate_ts : nullptr;
    T* y = (T*)a.y + p.b * a.T * D + p.base;
    const unsigned x_step = (unsigned)a.x_ts * kSize, dt_step = (unsigned)a.dt_ts * kSize, gate_step = (unsigned)a.gate_ts * kSize;
    BcTile<T, R> bc(a, p, p.t0, true, !ENDS);
    T xr[O], dr[O], gr[O];
    auto fetch = [&](int left) {                                          // rows behind the first `left` repeat the last
        bc.fetch(N, left);
        const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(x), 0, -1, 0x00020000);
        const auto rd = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(dt), 0, -1, 0x00020000);
        const auto rg = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(gate), 0, -1, 0x00020000);
#pragma unroll
        for (int j = 0; j < O; ++j) {
            const unsigned row = own + j < left ? own + j : left - 1, at = p.lane * kSize;
            xr[j] = buffer_get<T>(rx, row * x_step + at, 0);
            dr[j] = buffer_get<T>(rd, row * dt_step + at, 0);
            if (gate) gr[j] = buffer_get<T>(rg, row * gate_step + at, 0);
        }
    };
    if (p.t0 < p.t1) fetch(tile_left(p, p.t0));
    float A2[L], h[L], sum = 0.0f;
    const long segment = (p.b * pl.S + p.s) * R * D + n0 * D;
    load_decay<L>(a, d, A2, n0);
    auto first = [&](float (&v)[L], int N) {
#pragma unroll
        for (int n = 0; n < L; ++n) v[n] = !ENDS && n0 + n < N && a.state_in ? a.state_in[(p.b * D + d) * N + n0 + n] : 0.0f;
    };
    if (ENDS) first(h, N);
    else if (pl.joined) load_states<L>(E + segment, D, d, h);
    else fold_segments<L>(E + n0 * D, sd, R * D, D, d, p.b * pl.S, 0, p.s, 1, A2, h, N, first);
    const float skip = a.skip ? a.skip[d] : 0.0f, dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    float* saved = !ENDS && a.saved ? a.saved + (p.b * ((a.T + kTile - 1) / kTile) + p.t0 / kTile) * R * D + n0 * D : nullptr;
    int buf = 0;
    for (long t = p.t0; t < p.t1; t += kTile, buf ^= 1) {
        const int left = tile_left(p, t);
        float xv[O], gv[O], de_own[O], dx_own[O], de[kTile], dx[kTile], yv[kTile], out[O];
        bc.lay(lds[buf]);
#pragma unroll
        for (int j = 0; j < O; ++j) {
            const float raw = to_f(dr[j]) + dtb, s = a.softplus ? softplus_f(raw) : raw;
            xv[j] = to_f(xr[j]);
            gv[j] = gate ? to_f(gr[j]) : 1.0f;
            if (gate) gv[j] *= sigmoid_f(gv[j]);
            de_own[j] = own + j < left ? s : 0.0f;                        // (delta = 0 leaves every state as it is)
            dx_own[j] = own + j < left ? s * xv[j] : 0.0f;
        }
        if (t + kTile < p.t1) {
            x += kTile * a.x_ts; dt += kTile * a.dt_ts; gate += gate ? kTile * a.gate_ts : 0; bc.move(1);
            fetch(tile_left(p, t + kTile));
        }
        if (saved) {
            if (p.live) store_states<L>(saved, D, d, h);
            saved += R * D;
        }
        to_all<P>(de_own, de);
        to_all<P>(dx_own, dx);
        order();
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            float b[L], c[L], e[L], acc[2] = {};
            bc_row<L>(lds[buf] + i * 2 * R + n0, b);
            if constexpr (!ENDS) bc_row<L>(lds[buf] + i * 2 * R + R + n0, c);
            decays<L>(de[i], A2, e);
            if constexpr (ENDS) sum += de[i];
#pragma unroll
            for (int n = 0; n < L; ++n) {
                h[n] = __builtin_fmaf(e[n], h[n], dx[i] * b[n]);
                if constexpr (!ENDS) acc[n & 1] = __builtin_fmaf(c[n], h[n], acc[n & 1]);
            }
            yv[i] = acc[0] + acc[1];
        }
        if constexpr (ENDS) continue;
        sums_to_own<P>(yv, out);
        const auto ry = __builtin_amdgcn_make_buffer_rsrc(y + t * D, 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int j = 0; j < O; ++j) {
            const T o = from_f<T>(__builtin_fmaf(skip, xv[j], out[j]) * gv[j]);
            const unsigned at = p.live && own + j < left ? (unsigned)(own + j) * (unsigned)D * kSize + p.lane * kSize : 0xfffffff0u;
            if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, o), ry, (int)at, 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, o), ry, (int)at, 0, 0);
        }
    }
    if (!p.live) return;
    if constexpr (ENDS) {
        store_states<L>(E + segment, D, d, h);
        if (p.part == 0) sd[(p.b * pl.S + p.s) * D + d] = sum;
        return;
    }
    for (long t = (p.t0 > p.t1 ? p.t0 : p.t1) + p.part; t < p.tz; t += P) (y + t * D)[p.lane] = from_f<T>(0.0f);
    if (a.state_out && p.s == pl.S - 1)
#pragma unroll
        for (int n = 0; n < L; ++n)
            if (n0 + n < N) a.state_out[(p.b * D + d) * N + n0 + n] = h[n];
}

// Backwards: g = dy silu(gate), q_t = c_t g_t + exp(delta_{t+1} a) q_{t+1} is the gradient of h_t.
// First pass of a split one: the gradient of the state in front of a segment where none comes in from behind it.
template <typename T, int R>
__global__ void __launch_bounds__(64) ssm_bwd_ends_kernel(const vsv_ssm_desc a, const vsv_ssm_grads gr, const ScanPlan pl, float* __restrict__ E,
                                                          float* __restrict__ sd) {
    __shared__ alignas(16) float lds[2][kTile * 2 * R];
    const ScanPos p = scan_pos(a, pl, blockIdx.x, 1);
    const long D = a.D, d = p.base + p.lane;
    float A2[R], q[R] = {}, sum = 0.0f;
    load_decay<R>(a, d, A2);
    const float dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    const long tl = p.t0 + (p.t1 - 1 - p.t0) / kTile * kTile;              // the last tile
    const T *dt = (const T*)a.dt + p.b * a.dt_bs + p.base + tl * a.dt_ts, *dy = (const T*)gr.dy + p.b * gr.dy_bs + p.base + tl * gr.dy_ts;
    const T* gate = a.gate ? (const T*)a.gate + p.b * a.gate_bs + p.base + tl * a.gate_ts : nullptr;
    BcTile<T, R> bc(a, p, tl, false, true);
    T dr[kTile], gtr[kTile], yr[kTile];
    auto fetch = [&](int left) {
        bc.fetch(a.N, left);
        load_tile(dt, (int)(a.dt_ts * (long)sizeof(T)), p.lane, left, dr);
        load_tile(dy, (int)(gr.dy_ts * (long)sizeof(T)), p.lane, left, yr);
        if (gate) load_tile(gate, (int)(a.gate_ts * (long)sizeof(T)), p.lane, left, gtr);
    };
    if (p.t0 < p.t1) fetch(tile_left(p, tl));
    int buf = 0;
    for (long t = tl; t >= p.t0 && p.t0 < p.t1; t -= kTile, buf ^= 1) {
        const int left = tile_left(p, t);
        float raw[kTile], de[kTile], g[kTile];
        bc.lay(lds[buf]);
        tile_steps(dr, dtb, a.softplus, left, raw, de);
        tile_values(yr, left, g);
        if (gate) {
            float gv[kTile];
            tile_values(gtr, left, gv);
#pragma unroll
            for (int i = 0; i < kTile; ++i) g[i] *= gv[i] * sigmoid_f(gv[i]);
        }
        if (t > p.t0) {
            dt -= kTile * a.dt_ts; dy -= kTile * gr.dy_ts; gate -= gate ? kTile * a.gate_ts : 0; bc.move(-1);
            fetch(kTile);
        }
        order();
#pragma unroll
        for (int i = kTile - 1; i >= 0; --i) {
            float c[R], e[R];
            bc_row<R>(lds[buf] + i * 2 * R + R, c);
            decays<R>(de[i], A2, e);
            sum += de[i];
            order();
#pragma unroll
            for (int n = 0; n < R; ++n) q[n] = e[n] * __builtin_fmaf(c[n], g[i], q[n]);
            order();
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
        float r0, r1;
        swap32(v[j], v[j + NV / 2], r0, r1);
        v[j] = r0 + r1;
    }
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
        float r0, r1;
        swap16(v[j], v[j + NV / 4], r0, r1);
        v[j] = r0 + r1;
    }
    const int l = threadIdx.x;
    if constexpr (NV >= 8) halve<kRor8, NV / 8>(v, l & 8);
    if constexpr (NV >= 16) halve<kHalfMirror, NV / 16>(v, l & 4); else v[0] += dpp<kHalfMirror>(v[0]);
    if constexpr (NV >= 32) halve<kXor2, NV / 32>(v, l & 2); else v[0] += dpp<kXor2>(v[0]);
    return v[0] + dpp<kXor1>(v[0]);
}

// A tile at a time from the state saved in front of it: its states are computed again into registers, then q runs through
// them in reverse, four states at a time so that they fit.  The gradients of b and c are sums over channels: over the
// wave's 64 here, over the channel blocks in ssm_sums_kernel; those of a, skip and dt_bias sums over time: here, and over
// sequences and segments there too.  All in a fixed order.  4x2048x2048 bf16: 265 to 274 us, vector units at two waves a SIMD.
template <typename T, int R>
__global__ void __launch_bounds__(64, 2) ssm_bwd_kernel(const vsv_ssm_desc a, const vsv_ssm_grads gr, const ScanPlan pl, const float* __restrict__ E,
                                                        const float* __restrict__ sd, float* __restrict__ part_bc, float* __restrict__ part_p) {
    __shared__ alignas(16) float lds[2][kTile * 2 * R];
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
    const long Dg = D / a.G, blk = (p.base - p.g * Dg) / 64;
    float* bc = part_bc + (((blk * a.B + p.b) * a.T) * a.G + p.g) * (2 * R);
    const long bc_ts = a.G * 2 * R;
    float A2[R], q[R], dA[R] = {};
    load_decay<R>(a, d, A2);
    auto first = [&](float (&v)[R], int N) {
#pragma unroll
        for (int n = 0; n < R; ++n) v[n] = n < N && gr.d_state_out ? gr.d_state_out[(p.b * D + d) * N + n] : 0.0f;
    };
    if (pl.joined) load_states<R>(E + (p.b * pl.S + p.s) * R * D, D, d, q);
    else fold_segments<R>(E, sd, R * D, D, d, p.b * pl.S, pl.S - 1, p.s, -1, A2, q, N, first);
    if (!p.live) {
#pragma unroll
        for (int n = 0; n < R; ++n) q[n] = 0.0f;
    }
    const float skip = a.skip ? a.skip[d] : 0.0f, dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    float dskip = 0.0f, ddtb = 0.0f;
    BcTile<T, R> bct(a, p, tl, true, true);
    T xr[kTile], dr[kTile], gtr[kTile], yr[kTile];
    auto fetch = [&](int left) {
        bct.fetch(N, left);
        load_tile(x, (int)(a.x_ts * (long)sizeof(T)), p.lane, left, xr);
        load_tile(dt, (int)(a.dt_ts * (long)sizeof(T)), p.lane, left, dr);
        load_tile(dy, (int)(gr.dy_ts * (long)sizeof(T)), p.lane, left, yr);
        if (gate) load_tile(gate, (int)(a.gate_ts * (long)sizeof(T)), p.lane, left, gtr);
    };
    if (p.t0 < p.t1) fetch(tile_left(p, tl));
    int buf = 0;
    for (long t = tl; t >= p.t0 && p.t0 < p.t1; t -= kTile, buf ^= 1) {
        const int left = tile_left(p, t);
        float h0[R], xv[kTile], raw[kTile], de[kTile], g[kTile], dsl[kTile];
        bct.lay(lds[buf]);
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
            saved -= R * D; bct.move(-1);
            fetch(kTile);
        }
        float qb[kTile] = {}, dde[kTile] = {}, yv[kTile] = {};
#pragma unroll
        for (int n0 = 0; n0 < R; n0 += H) {
            float hs[kTile + 1][H];
#pragma unroll
            for (int n = 0; n < H; ++n) hs[0][n] = h0[n0 + n];
            order();
#pragma unroll
            for (int i = 0; i < kTile; ++i) {
                float b[H], e[H], dei = de[i];
                bc_row<H>(lds[buf] + i * 2 * R + n0, b);
                pin(dei);
                const float dx = dei * xv[i];
                decays<H>(dei, A2 + n0, e);
                order();
#pragma unroll
                for (int n = 0; n < H; ++n) {
                    hs[i + 1][n] = __builtin_fmaf(e[n], hs[i][n], dx * b[n]);
                    pin(hs[i + 1][n]);
                }
                order();
            }
#pragma unroll
            for (int i = kTile - 1; i >= 0; --i) {
                float b[H], c[H], e[H], v[2 * H], dei = de[i];
                bc_row<H>(lds[buf] + i * 2 * R + n0, b);
                bc_row<H>(lds[buf] + i * 2 * R + R + n0, c);
                pin(dei);
                const float dx = dei * xv[i];
                decays<H>(dei, A2 + n0, e);
                order();
#pragma unroll
                for (int n = 0; n < H; ++n) {
                    float& qn = q[n0 + n];
                    qn = __builtin_fmaf(c[n], g[i], qn);
                    yv[i] = __builtin_fmaf(c[n], hs[i + 1][n], yv[i]);
                    qb[i] = __builtin_fmaf(b[n], qn, qb[i]);
                    v[n] = qn * dx;
                    v[H + n] = g[i] * hs[i + 1][n];
                    qn *= e[n];
                    const float w = qn * hs[i][n];
                    dde[i] = __builtin_fmaf(A2[n0 + n], w, dde[i]);
                    dA[n0 + n] = __builtin_fmaf(dei, w, dA[n0 + n]);
                    pin(qn); pin(dA[n0 + n]);
                }
                pin(yv[i]); pin(qb[i]); pin(dde[i]);
                const float sum = wave_sums<2 * H>(v);
                constexpr int kEach = 64 / (2 * H);
                if (i < left && threadIdx.x % kEach == 0) {
                    const int j = threadIdx.x / kEach;                      // b's H states, then c's
                    bc[(t + i) * bc_ts + n0 + (j < H ? j : j - H + R)] = sum;
                }
                order();
            }
        }
        float dxv[kTile], ddv[kTile];
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            const float dd = __builtin_fmaf(xv[i], qb[i], dde[i] * (1.0f / kLog2e));
            ddv[i] = i < left ? (a.softplus ? dd * sigmoid_f(raw[i]) : dd) : 0.0f;
            dskip = __builtin_fmaf(g[i], xv[i], dskip);
            ddtb += ddv[i];
            dxv[i] = __builtin_fmaf(qb[i], de[i], g[i] * skip);
        }
        tile_store(dx_o + t * D, D, p, left, dxv);
        tile_store(ddt_o + t * D, D, p, left, ddv);
        if (gate) {
#pragma unroll
            for (int i = 0; i < kTile; ++i) yv[i] = dsl[i] * __builtin_fmaf(skip, xv[i], yv[i]);
            tile_store(dg_o + t * D, D, p, left, yv);
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

// The last sums of the backward pass, in a fixed order.  Workgroups below bc_blocks: db, dc from the channel blocks' shares
// (blocks, B T G, 2 R), rounded once; the others: da, dskip, d_dt_bias from the sequences' and segments' (rows, R + 2, D).
template <typename T>
__global__ void __launch_bounds__(256) ssm_sums_kernel(const float* __restrict__ part, long blocks, long bc_rows, unsigned bc_blocks, int R, int N,
                                                       T* __restrict__ db, T* __restrict__ dc, const float* __restrict__ part_p, long rows,
                                                       long D, float* __restrict__ da, float* __restrict__ dskip, float* __restrict__ ddtb) {
    __shared__ float red[4][64];
    if (blockIdx.x < bc_blocks) {
        const long id = (long)blockIdx.x * 256 + threadIdx.x, M = bc_rows * 2 * R;
        if (id >= M) return;
        const long r = id / (2 * R);
        const int j = (int)(id - r * 2 * R), n = j < R ? j : j - R;
        if (n >= N) return;
        float s = 0.0f;
#pragma unroll 8
        for (long k = 0; k < blocks; ++k) s += part[k * M + id];
        (j < R ? db : dc)[r * N + n] = from_f<T>(s);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long M = (R + 2) * D, m = (long)(blockIdx.x - bc_blocks) * 64 + lane;
    float s = 0.0f;
    if (m < M) {
#pragma unroll 8
        for (long r = wave; r < rows; r += 4) s += part_p[r * M + m];
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
// states as one access, and add up the output over the P lanes (1000x4096 bf16, 16 states: 100 us, 5.3 TB/s).  The other inputs
// are small, but each is a memory instruction of every wave: WIDE takes a lane's four values of b and c at once (one at a time:
// 136 us), and all are under way before the first is used.
template <typename T, int R, bool WIDE>
__global__ void __launch_bounds__(256) ssm_step_kernel(const vsv_ssm_desc a) {
    constexpr int P = R / 4;
    const long id = ((long)blockIdx.x * 256 + threadIdx.x) / P;
    const int part = threadIdx.x % P, n0 = part * 4;
    if (id >= a.B * a.D) return;                                          // (all P lanes of a channel leave together)
    const long b = id / a.D, d = id - b * a.D, g = d / (a.D / a.G);
    const int N = a.N;
    const T *bp = (const T*)a.b + b * a.b_bs + g * a.b_gs + n0, *cp = (const T*)a.c + b * a.c_bs + g * a.c_gs + n0;
    float* st = a.state_out + id * N + n0;
    const float* ap = a.a + d * N + n0;
    float h[4] = {}, av[4] = {}, bv[4] = {}, cv[4] = {};
    if (WIDE) { load_vec<float, 4>(st, h); load_vec<T, 4>(bp, bv); load_vec<T, 4>(cp, cv); load_vec<float, 4>(ap, av); }
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < N) { h[j] = st[j]; av[j] = ap[j]; bv[j] = to_f(bp[j]); cv[j] = to_f(cp[j]); }
    }
    const float xv = to_f(((const T*)a.x)[b * a.x_bs + d]), dtb = a.dt_bias ? a.dt_bias[d] : 0.0f;
    const float raw = to_f(((const T*)a.dt)[b * a.dt_bs + d]) + dtb;
    const float skip = a.skip ? a.skip[d] : 0.0f, gv = a.gate ? to_f(((const T*)a.gate)[b * a.gate_bs + d]) : 0.0f;
    const float de = a.softplus ? softplus_f(raw) : raw, dx = de * xv;
    float acc = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (!WIDE && n0 + j >= N) continue;
        h[j] = __builtin_fmaf(exp2_fast(de * av[j] * kLog2e), h[j], dx * bv[j]);
        acc = __builtin_fmaf(cv[j], h[j], acc);
    }
    if (WIDE) store_vec<float, 4>(st, h);
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < N) st[j] = h[j];
    }
#pragma unroll
    for (int o = 1; o < P; o <<= 1) acc += __shfl_xor(acc, o, 64);
    if (part) return;
    acc = __builtin_fmaf(skip, xv, acc);
    if (a.gate) acc *= gv * sigmoid_f(gv);
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

// Whether every row starts on a word of v elements.
bool conv_words(const vsv_short_conv_desc* a, const vsv_short_conv_grads* g, size_t size, long v) {
    bool ok = a->D % v == 0 && a->x_bs % v == 0 && a->x_ts % v == 0 && aligned(a->x, v * size) && aligned(a->y, v * size);
    if (g) ok = ok && g->dy_bs % v == 0 && g->dy_ts % v == 0 && aligned(g->dy, v * size) && aligned(g->dx, v * size);
    return ok;
}
// Channels per thread: four where the rows allow it (eight in 16 bits: forward 80 us for 67, backward the same 92 us).
int conv_vec(const vsv_short_conv_desc* a, const vsv_short_conv_grads* g) {
    const size_t size = a->dtype == VSV_F32 ? 4 : 2;
    return conv_words(a, g, size, 4) ? 4 : 1;
}

// Time steps per thread: the longer, the less is read twice and the fewer sums are left over, as long as the threads fill the
// chip.  Forward eight waves for every SIMD (8x2048x4096 bf16: four and eight 61 us); backward, where a chunk leaves K + 1 sums
// per channel, two (92 us and 4 for the sums; one 105 and 5, four 100 and 7).
constexpr long kConvFill = 524288, kConvBwdFill = 131072;
long conv_chunk(const vsv_short_conv_desc* a, long fill, long vec) {
    const long rows = a->B * (a->D / vec);
    long chunk = 16;
    while (chunk < 256 && rows * ((a->T + 2 * chunk - 1) / (2 * chunk)) >= fill) chunk *= 2;
    return chunk;
}
long conv_chunks(const vsv_short_conv_desc* a, long chunk) { return a->T > 0 ? (a->T + chunk - 1) / chunk : 1; }
// The backward pass's chunk goes by the sizes alone, so that its workspace does too.
long conv_bwd_chunk(const vsv_short_conv_desc* a) {
    return conv_chunk(a, kConvBwdFill, a->D % 4 == 0 ? 4 : 1);
}

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
    const long most = 0x7fffffffL / (4 * kTile);                          // (a tile's rows are addressed with 32 bits)
    if (a->D > most || (a->T > 1 && (a->x_ts > most || a->dt_ts > most || a->gate_ts > most || a->x_ts < 0 || a->dt_ts < 0 || a->gate_ts < 0))) {
        set_error("%s: more than %ld channels, or a time stride of more elements than that", what, most); return -2;
    }
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

// How the work is divided.  A split of time costs a second pass (1.8 times the work) and a launch, so it pays below about half
// a wave per SIMD (1024 of them): then as many segments as make two waves per SIMD, none shorter than two tiles (three were
// slower at 64x128x100 to 5x777x198), at most kMaxSegments (1x4096x256 forward and backward: 64 segments 173 us, 256 124).  A
// few segments are folded by those behind them, many in a launch of their own (5x777x198, 48 segments, forward: 34 and 31 us;
// 4x2048x2048, 16 segments, backward: 329 and 340).
//   Forward, below as many waves, a channel's states are shared by R / 4 lanes where the sequence is short or the work is little: below
// 64 steps, or up to kShareTiles tiles over all waves.  (It is a bound on work, not on waves: sharing issues 1.4 times the
// instructions, which costs nothing while SIMDs stand idle.  16x256x100: 21 us with one lane a channel, 15; 1x1024x256: 25 and 18;
// 64x1024x100, 16384 tiles: 74 and 96, both of them split; from 64 steps on sharing was not measured without a split.)  A sequence that
// is short enough is not split at all (64x60x100: in one pass 12, in segments 13; 64x96x100: 17 and 16.5).  From 512 waves on nothing is
// split or shared: 8x512x4096, 512 waves on 1024 SIMDs, takes 195 us, of which 24 cycles a state are 94 on the SIMDs
// that have a wave.
constexpr long kMaxSegments = 256, kSplitFrom = 40, kJoinFrom = 24, kShareBelow = 64, kShareTiles = 6144, kSplitWaves = 2048;

ScanPlan scan_plan(const vsv_ssm_desc* a, bool forward) {
    ScanPlan pl = {};
    const long waves = a->B * a->G * ssm_blocks(a), tiles = (a->T + kTile - 1) / kTile;
    long S = 1;
    pl.P = 1;
    if (waves > 0 && waves < 512) {
        if (forward && a->N > 4 && (a->T < kShareBelow || waves * tiles <= kShareTiles)) pl.P = padded_states(a->N) / 4;
        if (a->T >= (pl.P > 1 ? kShareBelow : kSplitFrom)) {
            S = (kSplitWaves + waves * pl.P - 1) / (waves * pl.P);
            if (S > tiles / 2) S = tiles / 2;
            if (S > kMaxSegments) S = kMaxSegments;
        }
    }
    const long per = tiles > 0 ? (tiles + S - 1) / S : 1;
    pl.seg = per * kTile;
    pl.S = tiles > 0 ? (int)((tiles + per - 1) / per) : 1;
    pl.joined = pl.S >= kJoinFrom;
    return pl;
}

size_t ends_floats(const vsv_ssm_desc* a, const ScanPlan& pl) {
    return pl.S > 1 ? (size_t)a->B * pl.S * (padded_states(a->N) + 1) * a->D : 0;
}
template <int R> int join_segments(const vsv_ssm_desc* a, const ScanPlan& pl, const float* init, bool back, float* E, const float* sd, hipStream_t stream) {
    if (!pl.joined) return 0;
    const long blocks = (a->B * R * a->D + 63) / 64;                      // (split scans have fewer than 512 waves of channels)
    hipLaunchKernelGGL(ssm_join_kernel<R>, dim3((unsigned)blocks), dim3(64), 0, stream, a->a, init, a->N, a->D, a->B, pl.S, back, E, sd);
    return op_launch_check("ssm_join_kernel");
}
size_t round4(size_t n) { return (n + 3) & ~(size_t)3; }

}  // namespace
}  // namespace vsv

using namespace vsv;

extern "C" int vsv_short_conv(const vsv_short_conv_desc* a, void* stream) {
    if (int rc = check_conv(a, "vsv_short_conv")) return rc;
    if (a->B == 0) return 0;
    const int vec = conv_vec(a, nullptr);
    const long chunk = conv_chunk(a, kConvFill, vec), nc = conv_chunks(a, chunk), nv = a->D / vec, blocks = (a->B * nc * nv + 255) / 256;
    if (blocks > kMaxBlocks) { set_error("vsv_short_conv: too many elements for one call"); return -2; }
    return by_dtype(a->dtype, "vsv_short_conv", [&](auto t) { return by_taps(a->K, [&](auto k) {
        using T = decltype(t);
        constexpr int K = decltype(k)::value;
        if (vec == 4) hipLaunchKernelGGL((short_conv_kernel<T, K, 4, 4>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, chunk, nc, nv);
        else hipLaunchKernelGGL((short_conv_kernel<T, K, 1, 4>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, chunk, nc, nv);
        return op_launch_check("short_conv_kernel");
    }); });
}

extern "C" size_t vsv_short_conv_backward_ws_bytes(const vsv_short_conv_desc* a) {
    if (check_conv(a, "vsv_short_conv_backward_ws_bytes")) return 0;
    return (size_t)a->B * conv_chunks(a, conv_bwd_chunk(a)) * (a->K + 1) * a->D * sizeof(float);
}

extern "C" int vsv_short_conv_backward(const vsv_short_conv_desc* a, const vsv_short_conv_grads* g, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_conv(a, "vsv_short_conv_backward")) return rc;
    if (!g || (a->B > 0 && a->T > 0 && (!g->dy || !g->dx))) { set_error("vsv_short_conv_backward: null pointer"); return -1; }
    if (ws_bytes < vsv_short_conv_backward_ws_bytes(a) || (a->B > 0 && (!ws || !aligned(ws, 16)))) {
        set_error("vsv_short_conv_backward: workspace too small or not on 16 bytes"); return -1;
    }
    const int vec = conv_vec(a, g);
    const long chunk = conv_bwd_chunk(a), nc = conv_chunks(a, chunk), nv = a->D / vec, M = (a->K + 1) * a->D, blocks = (a->B * nc * nv + 255) / 256;
    if (blocks > kMaxBlocks) { set_error("vsv_short_conv_backward: too many elements for one call"); return -2; }
    if (a->B > 0) {
        const int rc = by_dtype(a->dtype, "vsv_short_conv_backward", [&](auto t) { return by_taps(a->K, [&](auto k) {
            using T = decltype(t);
            constexpr int K = decltype(k)::value;
            if (vec == 4) hipLaunchKernelGGL((short_conv_bwd_kernel<T, K, 4, 4>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, *g, chunk, nc, nv, (float*)ws);
            else hipLaunchKernelGGL((short_conv_bwd_kernel<T, K, 1, 4>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a, *g, chunk, nc, nv, (float*)ws);
            return op_launch_check("short_conv_bwd_kernel");
        }); });
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
    return ends_floats(a, scan_plan(a, true)) * sizeof(float);
}

extern "C" int vsv_ssm_scan(const vsv_ssm_desc* a, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_ssm(a, "vsv_ssm_scan")) return rc;
    if (a->B == 0) return 0;
    const size_t need = vsv_ssm_scan_ws_bytes(a);
    if (ws_bytes < need || (need && !aligned(ws, 16)) || (need && !ws)) { set_error("vsv_ssm_scan: workspace too small or not on 16 bytes"); return -1; }
    if (a->saved && !aligned(a->saved, 16)) { set_error("vsv_ssm_scan: saved must be on 16 bytes"); return -1; }
    const ScanPlan pl = scan_plan(a, true);
    const long waves = a->B * a->G * ssm_blocks(a);
    if (waves > kMaxBlocks / pl.S) { set_error("vsv_ssm_scan: too many sequences and channels for one call"); return -2; }
    float *E = (float*)ws, *sd = E + (size_t)a->B * pl.S * padded_states(a->N) * a->D;
    return by_dtype(a->dtype, "vsv_ssm_scan", [&](auto t) { return by_states(a->N, [&](auto r) {
        using T = decltype(t);
        constexpr int R = decltype(r)::value;
        if constexpr (R > 4) {
            if (pl.P > 1) {
                constexpr int P = R / 4, kCh = 64 / P;
                const long groups = a->B * a->G * ((a->D / a->G + kCh - 1) / kCh);
                if (pl.S > 1) {
                    hipLaunchKernelGGL((ssm_shared_kernel<T, R, P, true>), dim3((unsigned)(groups * (pl.S - 1))), dim3(64), 0, (hipStream_t)stream, *a, pl, E, sd);
                    if (int rc = op_launch_check("ssm_shared_kernel")) return rc;
                    if (int rc = join_segments<R>(a, pl, a->state_in, false, E, sd, (hipStream_t)stream)) return rc;
                }
                hipLaunchKernelGGL((ssm_shared_kernel<T, R, P, false>), dim3((unsigned)(groups * pl.S)), dim3(64), 0, (hipStream_t)stream, *a, pl, E, sd);
                return op_launch_check("ssm_shared_kernel");
            }
        }
        if (pl.S > 1) {
            hipLaunchKernelGGL((ssm_ends_kernel<T, R>), dim3((unsigned)(waves * (pl.S - 1))), dim3(64), 0, (hipStream_t)stream, *a, pl, E, sd);
            if (int rc = op_launch_check("ssm_ends_kernel")) return rc;
            if (int rc = join_segments<R>(a, pl, a->state_in, false, E, sd, (hipStream_t)stream)) return rc;
        }
        hipLaunchKernelGGL((ssm_scan_kernel<T, R>), dim3((unsigned)(waves * pl.S)), dim3(64), 0, (hipStream_t)stream, *a, pl, E, sd);
        return op_launch_check("ssm_scan_kernel");
    }); });
}

namespace {
size_t part_bc_floats(const vsv_ssm_desc* a) { return (size_t)ssm_blocks(a) * a->B * a->T * a->G * 2 * padded_states(a->N); }
}  // namespace

extern "C" size_t vsv_ssm_scan_backward_ws_bytes(const vsv_ssm_desc* a) {
    if (check_ssm(a, "vsv_ssm_scan_backward_ws_bytes")) return 0;
    const ScanPlan pl = scan_plan(a, false);
    return (round4(ends_floats(a, pl)) + round4(part_bc_floats(a)) +
            (size_t)a->B * pl.S * (padded_states(a->N) + 2) * a->D) * sizeof(float);
}

extern "C" int vsv_ssm_scan_backward(const vsv_ssm_desc* a, const vsv_ssm_grads* g, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_ssm(a, "vsv_ssm_scan_backward")) return rc;
    if (!g || (a->B > 0 && a->T > 0 && (!a->saved || !g->dy || !g->dx || !g->ddt || !g->db || !g->dc || (a->gate && !g->dgate)))) {
        set_error("vsv_ssm_scan_backward: null pointer"); return -1;
    }
    if (a->T > 1 && (g->dy_ts < 0 || g->dy_ts > 0x7fffffffL / (4 * kTile))) { set_error("vsv_ssm_scan_backward: bad time stride of dy"); return -2; }
    if (ws_bytes < vsv_ssm_scan_backward_ws_bytes(a) || (a->B > 0 && (!ws || !aligned(ws, 16)))) {
        set_error("vsv_ssm_scan_backward: workspace too small or not on 16 bytes"); return -1;
    }
    if (a->saved && !aligned(a->saved, 16)) { set_error("vsv_ssm_scan_backward: saved must be on 16 bytes"); return -1; }
    const ScanPlan pl = scan_plan(a, false);
    const int R0 = padded_states(a->N);
    const long nb = ssm_blocks(a), waves = a->B * a->G * nb, rows = a->B * a->T * a->G;
    if (waves > kMaxBlocks / pl.S) { set_error("vsv_ssm_scan_backward: too many elements for one call"); return -2; }
    float *E = (float*)ws, *sd = E + (size_t)a->B * pl.S * R0 * a->D;
    float *pbc = E + round4(ends_floats(a, pl)), *pp = pbc + round4(part_bc_floats(a));
    if (a->B > 0) {
        const int rc = by_dtype(a->dtype, "vsv_ssm_scan_backward", [&](auto t) { return by_states(a->N, [&](auto r) {
            using T = decltype(t);
            constexpr int R = decltype(r)::value;
            if (pl.S > 1) {
                hipLaunchKernelGGL((ssm_bwd_ends_kernel<T, R>), dim3((unsigned)(waves * (pl.S - 1))), dim3(64), 0, (hipStream_t)stream, *a, *g, pl, E, sd);
                if (int rc = op_launch_check("ssm_bwd_ends_kernel")) return rc;
                if (int rc = join_segments<R>(a, pl, g->d_state_out, true, E, sd, (hipStream_t)stream)) return rc;
            }
            hipLaunchKernelGGL((ssm_bwd_kernel<T, R>), dim3((unsigned)(waves * pl.S)), dim3(64), 0, (hipStream_t)stream, *a, *g, pl, E, sd, pbc, pp);
            return op_launch_check("ssm_bwd_kernel");
        }); });
        if (rc) return rc;
    }
    const long bc_blocks = (rows * 2 * R0 + 255) / 256, blocks = bc_blocks + ((R0 + 2) * a->D + 63) / 64;
    if (blocks > kMaxBlocks) { set_error("vsv_ssm_scan_backward: too many elements for one call"); return -2; }
    return by_dtype(a->dtype, "vsv_ssm_scan_backward", [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(ssm_sums_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, pbc, nb, rows, (unsigned)bc_blocks, R0, a->N,
                           (T*)g->db, (T*)g->dc, pp, a->B * pl.S, a->D, g->da, g->dskip, g->ddt_bias);
        return op_launch_check("ssm_sums_kernel");
    });
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
            const long w = 4 * (long)sizeof(T);
            if (a->N == RR && aligned(a->state_out, 16) && aligned(a->a, 16) && aligned(a->b, w) && aligned(a->c, w) &&
                a->b_bs % 4 == 0 && a->b_gs % 4 == 0 && a->c_bs % 4 == 0 && a->c_gs % 4 == 0)
                hipLaunchKernelGGL((ssm_step_kernel<T, RR, true>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a);
            else
                hipLaunchKernelGGL((ssm_step_kernel<T, RR, false>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a);
            return op_launch_check("ssm_step_kernel");
        });
    });
}
