// AdamW over many tensors in one launch, moments held in 32 bits or in 8.
//   p *= 1 - lr wd;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
//   p -= lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Every value is read once and written once and little is computed: bound by memory.  The tensors' addresses travel in
// the launch's arguments, so there is no table in device memory to keep or to copy, and nothing to look up on replay.
#include <cfloat>
#include <cmath>

#include "vsv_ops.h"

namespace vsv {
namespace {

constexpr int kMaxTensors = 60;      // per launch: the argument block stays below 4 KiB
constexpr int kBlock8 = VSV_ADAMW_BLOCK;

struct Hyper {
    float decay, b1, w1, b2, w2, eps, rate, root, inv_root;
    double b1d, w1d, b2d, w2d;
    unsigned dither;
};
struct Table {
    vsv_adamw_tensor t[kMaxTensors];
    unsigned first[kMaxTensors + 1]; // first workgroup of each tensor
    int n;
};

__device__ inline int tensor_of(const Table& tab, unsigned blk) {
    int lo = 0, hi = tab.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= blk) lo = mid; else hi = mid;
    }
    return lo;
}

// ---- 32 bits -----------------------------------------------------------------------------------------------------
// 168 M float32 parameters: 883 us, 5.3 TB/s.  Eight elements a thread, all loads ahead.
constexpr int kPer32 = 4, kIter32 = 2, kChunk32 = 256 * kPer32 * kIter32;

__device__ inline void update32(float& p, float g, float& m, float& v, const Hyper& h) {
    m = __builtin_fmaf(h.b1, m, h.w1 * g);
    v = __builtin_fmaf(h.b2, v, h.w2 * g * g);
    p = p * h.decay - h.rate * m / (sqrtf(v) / h.root + h.eps);
}

template <typename T>
__global__ void __launch_bounds__(256) adamw32_kernel(const Table tab, const Hyper h) {
    const int ti = tensor_of(tab, blockIdx.x);
    const vsv_adamw_tensor& e = tab.t[ti];
    const long base = (long)(blockIdx.x - tab.first[ti]) * kChunk32;
    T* p = (T*)e.p; const T* g = (const T*)e.g; float *m = (float*)e.m, *v = (float*)e.v;
    const bool wide = (((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) == 0 && (((uintptr_t)m | (uintptr_t)v) & 15) == 0;
    if (wide && base + kChunk32 <= e.n) {
        float pv[kIter32][4], gv[kIter32][4], mv[kIter32][4], vv[kIter32][4];
#pragma unroll
        for (int i = 0; i < kIter32; ++i) {
            const long o = base + (i * 256 + threadIdx.x) * 4;
            load_vec<T, 4>(p + o, pv[i]); load_vec<T, 4>(g + o, gv[i]);
            load_vec<float, 4>(m + o, mv[i]); load_vec<float, 4>(v + o, vv[i]);
        }
#pragma unroll
        for (int i = 0; i < kIter32; ++i) {
            const long o = base + (i * 256 + threadIdx.x) * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) update32(pv[i][j], gv[i][j], mv[i][j], vv[i][j], h);
            store_vec<T, 4>(p + o, pv[i]);
            store_vec<float, 4>(m + o, mv[i]); store_vec<float, 4>(v + o, vv[i]);
        }
        return;
    }
    for (long o = base + threadIdx.x; o < e.n && o < base + kChunk32; o += 256) {
        float pv = to_f(p[o]), mv = m[o], vv = v[o];
        update32(pv, to_f(g[o]), mv, vv, h);
        p[o] = from_f<T>(pv); m[o] = mv; v[o] = vv;
    }
}

// ---- 8 bits ------------------------------------------------------------------------------------------------------
// Blocks of 256 elements share two float32 scales, max |m| and max v.  A code k of m stands for sign s (k/127)^2, one of v
// for s (k/255)^4: steps grow with the value, so m spans 4 and v 9 orders of magnitude below a block's largest.
//   Rounding: of the two codes around a value the upper one where the value is more than a share u of the way, u from an
// additive (Weyl) sequence over steps and elements (for v, 1 - u).  Over steps u is spread evenly, so the rounding is
// unbiased in time; to the nearest code, v would never move: beta2 = 0.999 changes it by 0.1 % a step, codes are at least
// 1.6 % apart.  v > 0 never becomes 0, which would leave m without its divisor.
//   168 M bf16 parameters: 417 to 461 us, the issue of 90 vector operations an element (its 10.06 bytes an element, 1.69 GB,
// take 350 us at the copy rate).
//   The moments are computed in 64 bits (full rate on this chip), and so is the choice of a code wherever float32 could
// choose another: the codes are the definition's, not a rounding away from it.
//   A gradient that is not finite leaves its element's moments alone and makes the parameter NaN: a NaN scale would take
// the other 255 elements along.
constexpr double kFullM = 127.0 * 127.0, kFullV = 255.0 * 255.0 * 255.0 * 255.0;
constexpr int kPer8 = 8, kLanes8 = kBlock8 / kPer8, kChunk8 = 256 * kPer8;

// (the float32 nearest to it: the moments that a step starts from are the ones that vsv_adamw_read8 shows; a scale comes
// divided by the full code's power)
__device__ inline float read_m8(int k, double s) { const float f = (float)k; return (float)((double)(f * __builtin_fabsf(f)) * s); }
__device__ inline float read_v8(unsigned k, double s) {
    const float f = (float)k;
    const double k2 = (double)(f * f);
    return (float)(k2 * k2 * s);
}

// The moments as the formulas write them, operation by operation: gradients of 16 bits have so few mantissas that a sum next
// to the middle between two float32 scales is no rarity, and a fused sum fell on the other side of it in 0.8 % of the blocks.
__device__ inline double next_m(double m, double g, const Hyper& h) {
#pragma clang fp contract(off)
    return m * h.b1d + g * h.w1d;
}
__device__ inline double next_v(double v, double g, const Hyper& h) {
#pragma clang fp contract(off)
    return v * h.b2d + g * g * h.w2d;
}

// The codes by the definition, in 64 bits.
__device__ inline int exact_m8(double x, double scale, double u) {
    const double y = fmin(fabs(x) / scale * kFullM, kFullM);
    double k = (double)(int)__builtin_amdgcn_sqrtf((float)y);
    if (k * k > y) k -= 1.0;
    if ((k + 1.0) * (k + 1.0) <= y) k += 1.0;
    return (int)k + (y - k * k > u * (2.0 * k + 1.0));
}
__device__ inline int exact_v8(double x, double scale, double u) {
    const double y = fmin(x / scale * kFullV, kFullV);
    double k = (double)(int)__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)y));
    double k2 = k * k, up = (k + 1.0) * (k + 1.0);
    if (k2 * k2 > y) { up = k2; k -= 1.0; k2 = k * k; }
    if (up * up <= y) { k2 = up; k += 1.0; up = (k + 1.0) * (k + 1.0); }
    return (int)k + (y - k2 * k2 > u * (up * up - k2 * k2));
}
// The same in float32 (a code as a float), where no more than 3e-5 of a gap is lost: `least` is the smallest distance to a
// threshold, in gaps less kNear, and the 64-bit form decides where it is negative.  Next to a code's own value k may come out
// one off, the share of the gap then next to 1 for next to 0 or the other way round: the code is the same for any u but those
// next to 0 and 1, which the caller counts as near.
constexpr float kNear = 1e-4f;
__device__ inline float step_up(float over) { return __builtin_amdgcn_fmed3f(over * 1e30f, 0.0f, 1.0f); }
__device__ inline float code_m8(float x, float inv, float u, float& least) {
    const float y = __builtin_fabsf(x) * inv, k = floorf(__builtin_amdgcn_sqrtf(y));
    const float gap = __builtin_fmaf(2.0f, k, 1.0f), over = __builtin_fmaf(-u, gap, __builtin_fmaf(-k, k, y));
    least = __builtin_fminf(least, __builtin_fmaf(-kNear, gap, __builtin_fabsf(over)));
    return k + step_up(over);
}
__device__ inline float code_v8(float x, float inv, float u, float& least) {
    const float y = x * inv, k = floorf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(y))), k2 = k * k;
    const float d = __builtin_fmaf(2.0f, k, 1.0f), gap = d * __builtin_fmaf(2.0f, k2, d);         // (k+1)^4 - k^4
    const float over = __builtin_fmaf(-u, gap, __builtin_fmaf(-k2, k2, y));
    least = __builtin_fminf(least, __builtin_fmaf(-kNear, gap, __builtin_fabsf(over)));
    return k + step_up(over);
}

// The largest of the 32 lanes that share a block.
template <int CTRL> __device__ inline float max_dpp(float v) {
    return __builtin_fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)));
}
__device__ inline float block_max(float v) {
    v = max_dpp<0xb1>(v);                                                 // lanes 1, 2, 7 - l, 15 - l apart
    v = max_dpp<0x4e>(v);
    v = max_dpp<0x141>(v);
    v = max_dpp<0x140>(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned r0 = r[0], r1 = r[1];                                  // and the neighbouring sixteen
    return __builtin_fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}

template <typename T>
__global__ void __launch_bounds__(256) adamw8_kernel(const Table tab, const Hyper h) {
    const int ti = tensor_of(tab, blockIdx.x);
    const vsv_adamw_tensor& e = tab.t[ti];
    const long o = (long)(blockIdx.x - tab.first[ti]) * kChunk8 + (long)threadIdx.x * kPer8;
    const long blk = o / kBlock8;
    if (blk * kBlock8 >= e.n) return;                                     // (a block's 32 lanes leave together)
    T* p = (T*)e.p; const T* g = (const T*)e.g; int8_t* mc = (int8_t*)e.m; uint8_t* vc = (uint8_t*)e.v;
    const bool wide = o + kPer8 <= e.n && (((uintptr_t)p | (uintptr_t)g) & 15) == 0 && (((uintptr_t)mc | (uintptr_t)vc) & 7) == 0;
    const int cnt = o >= e.n ? 0 : e.n - o < kPer8 ? (int)(e.n - o) : kPer8;
    float pv[kPer8] = {}, gv[kPer8] = {};
    Pack<int8_t, kPer8> mk = {};
    Pack<uint8_t, kPer8> vk = {};
    if (wide) {
        load_vec<T, kPer8>(p + o, pv); load_vec<T, kPer8>(g + o, gv);
        mk = *(const Pack<int8_t, kPer8>*)(mc + o);
        vk = *(const Pack<uint8_t, kPer8>*)(vc + o);
    } else {
#pragma unroll
        for (int j = 0; j < kPer8; ++j)
            if (j < cnt) { pv[j] = to_f(p[o + j]); gv[j] = to_f(g[o + j]); mk.v[j] = mc[o + j]; vk.v[j] = vc[o + j]; }
    }
    const double ms = (double)e.m_scale[blk] * (1.0 / kFullM), vs = (double)e.v_scale[blk] * (1.0 / kFullV);
    double m[kPer8], v[kPer8];
    float finite = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer8; ++j) {
        const double gd = gv[j];
        m[j] = next_m(read_m8(mk.v[j], ms), gd, h);
        v[j] = next_v(read_v8(vk.v[j], vs), gd, h);
        finite = __builtin_fmaf(gv[j], 0.0f, finite);
    }
    if (finite != 0.0f) {                                                 // some gradient here is not finite
        asm volatile("");                                                 // (a branch: the selects would cost every step six operations an element)
#pragma unroll
        for (int j = 0; j < kPer8; ++j)
            if (!__builtin_isfinite(gv[j])) { m[j] = read_m8(mk.v[j], ms); v[j] = read_v8(vk.v[j], vs); pv[j] = __builtin_nanf(""); }
    }
    // (the largest of the values rounded to float32 is the largest value rounded)
    float m32[kPer8], v32[kPer8], sm = 0.0f, sv = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer8; ++j) {
        m32[j] = (float)m[j];
        v32[j] = (float)v[j];
        sm = __builtin_fmaxf(sm, __builtin_fabsf(m32[j]));
        sv = __builtin_fmaxf(sv, v32[j]);
    }
    // (the fast root and reciprocal, an ulp each; without an eps subnormal second moments would count, which they lose)
    if (h.eps >= 1e-15f) {
#pragma unroll
        for (int j = 0; j < kPer8; ++j)
            pv[j] = __builtin_fmaf(-h.rate * m32[j], __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_amdgcn_sqrtf(v32[j]), h.inv_root, h.eps)),
                                   pv[j] * h.decay);
    } else {
        asm volatile("");
#pragma unroll
        for (int j = 0; j < kPer8; ++j) pv[j] = pv[j] * h.decay - h.rate * (float)(m[j] / (sqrt(v[j]) * h.inv_root + h.eps));
    }
    sm = __builtin_fminf(block_max(sm), FLT_MAX);
    sv = __builtin_fminf(block_max(sv), FLT_MAX);
    // (float32 holds neither factor where the scale is next to its limits: there, all codes by the definition)
    const bool plain = (sm > 0.0f && (sm < 1e-30f || sm > 1e30f)) || (sv > 0.0f && (sv < 1e-26f || sv > 1e30f));
    const float im = sm > 0.0f ? (float)kFullM * __builtin_amdgcn_rcpf(sm) : 0.0f, iv = sv > 0.0f ? (float)kFullV * __builtin_amdgcn_rcpf(sv) : 0.0f;
    const unsigned some = sv > 0.0f;
#pragma unroll
    for (int j = 0; j < kPer8; ++j) {
        const unsigned weyl = (unsigned)(o + j) * VSV_ADAMW_WEYL_I + h.dither;
        const float u = (float)weyl * 0x1p-32f;
        float least = plain ? -1.0f : 0.5f - kNear - __builtin_fabsf(u - 0.5f);
        const float km = code_m8(m32[j], im, u, least), kv = code_v8(v32[j], iv, 1.0f - u, least);
        int cm = (int)__builtin_copysignf(km, m32[j]), cv = (int)kv;
        if (!(least >= 0.0f)) {
            const double ud = ((double)weyl + 0.5) * 0x1p-32;
            cm = sm > 0.0f ? exact_m8(m[j], sm, ud) : 0;
            cm = m[j] < 0.0 ? -cm : cm;
            cv = sv > 0.0f ? exact_v8(v[j], sv, 1.0 - ud) : 0;
        }
        // v > 0 (its upper word, then, is not 0) never gets code 0
        const unsigned high = (unsigned)(__builtin_bit_cast(unsigned long long, v[j]) >> 32), one = high < some ? high : some;
        mk.v[j] = (int8_t)cm;
        vk.v[j] = (uint8_t)((unsigned)cv > one ? (unsigned)cv : one);
    }
    if (wide) {
        store_vec<T, kPer8>(p + o, pv);
        *(Pack<int8_t, kPer8>*)(mc + o) = mk;
        *(Pack<uint8_t, kPer8>*)(vc + o) = vk;
    } else {
#pragma unroll
        for (int j = 0; j < kPer8; ++j)
            if (j < cnt) { p[o + j] = from_f<T>(pv[j]); mc[o + j] = mk.v[j]; vc[o + j] = vk.v[j]; }
    }
    if (threadIdx.x % kLanes8 == 0) { e.m_scale[blk] = sm; e.v_scale[blk] = sv; }
}

// The values that the codes stand for, in float32: t.p and t.g are the two outputs here (four fifths of its bytes are writes:
// 168 M elements 240 to 340 us).
__global__ void __launch_bounds__(256) adamw8_read_kernel(const Table tab) {
    const int ti = tensor_of(tab, blockIdx.x);
    const vsv_adamw_tensor& e = tab.t[ti];
    const long o = (long)(blockIdx.x - tab.first[ti]) * kChunk8 + (long)threadIdx.x * kPer8;
    if (o >= e.n) return;
    const int8_t* mc = (const int8_t*)e.m; const uint8_t* vc = (const uint8_t*)e.v;
    float *mo = (float*)e.p, *vo = (float*)e.g;
    const double ms = (double)e.m_scale[o / kBlock8] * (1.0 / kFullM), vs = (double)e.v_scale[o / kBlock8] * (1.0 / kFullV);
    if (o + kPer8 <= e.n && (((uintptr_t)mo | (uintptr_t)vo) & 15) == 0 && (((uintptr_t)mc | (uintptr_t)vc) & 7) == 0) {
        const auto mk = *(const Pack<int8_t, kPer8>*)(mc + o);
        const auto vk = *(const Pack<uint8_t, kPer8>*)(vc + o);
#pragma unroll
        for (int half = 0; half < kPer8; half += 4) {
            float m[4], v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { m[j] = read_m8(mk.v[half + j], ms); v[j] = read_v8(vk.v[half + j], vs); }
            store_vec<float, 4>(mo + o + half, m);
            store_vec<float, 4>(vo + o + half, v);
        }
        return;
    }
    for (int j = 0; j < kPer8 && o + j < e.n; ++j) { mo[o + j] = read_m8(mc[o + j], ms); vo[o + j] = read_v8(vc[o + j], vs); }
}

// Launches f(table, workgroups) for every kMaxTensors tensors.
template <typename F> int over_tables(const vsv_adamw_tensor* t, int n, long chunk, const char* what, F&& f) {
    for (int at = 0; at < n;) {
        Table tab;
        tab.n = 0;
        long blocks = 0;
        while (at < n && tab.n < kMaxTensors) {
            const long b = (t[at].n + chunk - 1) / chunk;
            if (b > 0x7fffffffL) { set_error("%s: tensor %d is too large", what, at); return -2; }
            if (blocks + b > 0x7fffffffL) break;
            if (b > 0) {
                tab.t[tab.n] = t[at];
                tab.first[tab.n++] = (unsigned)blocks;
                blocks += b;
            }
            ++at;
        }
        if (!blocks) continue;
        tab.first[tab.n] = (unsigned)blocks;
        f(tab, (unsigned)blocks);
        if (int rc = op_launch_check(what)) return rc;
    }
    return 0;
}

int check_tensors(const vsv_adamw_tensor* t, int n, int bits, const char* what) {
    if (n < 0 || (n > 0 && !t)) { set_error("%s: null table", what); return -1; }
    if (bits != 8 && bits != 32) { set_error("%s: moments are held in 8 or 32 bits, not %d", what, bits); return -1; }
    for (int i = 0; i < n; ++i) {
        if (t[i].n < 0) { set_error("%s: tensor %d has a negative size", what, i); return -1; }
        if (t[i].n > 0 && (!t[i].p || !t[i].g || !t[i].m || !t[i].v || (bits == 8 && (!t[i].m_scale || !t[i].v_scale)))) {
            set_error("%s: tensor %d has a null pointer", what, i); return -1;
        }
    }
    return 0;
}

}  // namespace
}  // namespace vsv

using namespace vsv;

extern "C" int vsv_adamw_multi(const vsv_adamw_tensor* tensors, int n_tensors, int dtype, int bits, double lr, double beta1, double beta2,
                               double eps, double weight_decay, long step, void* stream) {
    if (int rc = check_tensors(tensors, n_tensors, bits, "vsv_adamw_multi")) return rc;
    if (step < 1) { set_error("vsv_adamw_multi: step counts from 1"); return -1; }
    if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0)) {
        set_error("vsv_adamw_multi: bad hyper-parameters"); return -1;
    }
    Hyper h;
    h.decay = (float)(1.0 - lr * weight_decay);
    h.b1 = (float)beta1; h.w1 = (float)(1.0 - beta1); h.b2 = (float)beta2; h.w2 = (float)(1.0 - beta2);
    h.eps = (float)eps;
    h.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    h.root = (float)std::sqrt(1.0 - std::pow(beta2, (double)step));
    h.inv_root = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    h.b1d = beta1; h.w1d = 1.0 - beta1; h.b2d = beta2; h.w2d = 1.0 - beta2;
    h.dither = (unsigned)step * VSV_ADAMW_WEYL_T;
    return by_dtype(dtype, "vsv_adamw_multi", [&](auto t) {
        using T = decltype(t);
        return over_tables(tensors, n_tensors, bits == 8 ? kChunk8 : kChunk32, "vsv_adamw_multi", [&](const Table& tab, unsigned blocks) {
            if (bits == 8) hipLaunchKernelGGL(adamw8_kernel<T>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tab, h);
            else hipLaunchKernelGGL(adamw32_kernel<T>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tab, h);
        });
    });
}

extern "C" int vsv_adamw_read8(const vsv_adamw_tensor* tensors, int n_tensors, void* stream) {
    if (int rc = check_tensors(tensors, n_tensors, 8, "vsv_adamw_read8")) return rc;
    return over_tables(tensors, n_tensors, kChunk8, "vsv_adamw_read8", [&](const Table& tab, unsigned blocks) {
        hipLaunchKernelGGL(adamw8_read_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, tab);
    });
}
