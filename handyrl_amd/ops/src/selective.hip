// Short causal convolution and selective state space scan over windows of
// steps, and their single-step forms.
//
// Convolution over the OBSERVED steps (u: the carried inputs, then x):
//   y_t = act(bias + sum_k w_k u_{t-K+1+k})
// Scan, per channel c and state n, with d = softplus(dt + dt_bias):
//   h_t = exp(d_t A) h_{t-1} + d_t B_t x_t,   y_t = (C_t . h_t + D x_t) silu(z_t)
// Steps whose mask is 0 leave the carried state as it is and give y = 0;
// nothing of what they hold is used.

#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <hip/hip_runtime.h>
#include "guards.h"

namespace {

using bf16 = __hip_bfloat16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16(v); }

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float* out) {
    const Pack<T, V> raw = *(const Pack<T, V>*)p;
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_float(raw.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float* in) {
    Pack<T, V> raw;
#pragma unroll
    for (int i = 0; i < V; ++i) raw.v[i] = from_float<T>(in[i]);
    *(Pack<T, V>*)p = raw;
}

// Four values of which the first `n` exist; the others read as 0.  `whole`, the
// same for all lanes, says that all four do and lie aligned.
template <typename T>
__device__ __forceinline__ Pack<T, 4> load_raw(const T* p, int n, bool whole) {
    if (whole) return *(const Pack<T, 4>*)p;
    Pack<T, 4> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = i < n ? p[i] : from_float<T>(0.f);
    return r;
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, int n, bool whole, float* out) {
    if (whole) {
        load_pack<T, 4>(p, out);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = i < n ? to_float(p[i]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int n, bool whole, const float* in) {
    if (whole) {
        store_pack<T, 4>(p, in);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = from_float<T>(in[i]);
    }
}

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.f + exp2_fast(-kLog2e * v));
}
// max(v, 0) + log1p(e), e = e^-|v|.  log1p(e) / e over [0, 1] as a polynomial of
// degree 8, fitted to the least largest relative error: 3.0e-8, and 2.0e-7 with
// the roundings of its evaluation.  Several of these stand beside every 16 steps
// of a scan, so their length counts.
__device__ __forceinline__ float softplus(float v) {
    const float e = exp2_fast(-kLog2e * fabsf(v));
    float p = 0.005232484545558691f;
    p = fmaf(p, e, -0.029504399746656418f);
    p = fmaf(p, e, 0.07822458446025848f);
    p = fmaf(p, e, -0.1366313099861145f);
    p = fmaf(p, e, 0.19105952978134155f);
    p = fmaf(p, e, -0.24842968583106995f);
    p = fmaf(p, e, 0.3331909477710724f);
    p = fmaf(p, e, -0.4999949336051941f);
    p = fmaf(p, e, 0.9999999403953552f);
    return fmaf(p, e, fmaxf(v, 0.f));
}

// ------------------------------------------------------------ convolution

struct ConvArgs {
    const void* x;              // (B, T, D), last axis dense
    const float* w;             // (D, K)
    const float* bias;          // (D) or null
    const void* state;          // (B, K-1, D) dense, or null: zeros
    const bool* mask;           // (B, T) or null
    const void* dy;             // (B, T, D) dense
    const void* dlast;          // (B, K-1, D) dense, or null
    void* y;                    // (B, T, D); backward: dx
    void* last;                 // (B, K-1, D); backward: dstate, or null
    float* parts;               // backward: (nparts, K+1, D)
    long batch, steps, xb, xt;
    int width, tile, tiles, nparts, silu;
};

// The masks of the 64 steps from `from` on as bits; 0 for steps outside [0, steps).
// The product gathers the low bits of eight bytes into one without a carry (a
// byte that was never a bool must not become another step's bit).
__device__ __forceinline__ unsigned long long seen_64(const bool* mask, long from, long steps) {
    unsigned long long bits = 0;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        const long t = from + 8 * g;
        unsigned long long w = 0;
        if (t >= 0 && t + 8 <= steps) {
            __builtin_memcpy(&w, mask + t, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (t + i >= 0 && t + i < steps) w |= (unsigned long long)mask[t + i] << (8 * i);
        }
        w &= 0x0101010101010101ull;
        bits |= ((w * 0x0102040810204080ull) >> 56) << (8 * g);
    }
    return bits;
}

// The last K-1 observed inputs before t0, oldest first.
template <typename T, int K, int V, bool MASKED>
__device__ __forceinline__ void conv_behind(const ConvArgs& p, long b, long t0, int c,
                                            float (&win)[K - 1][V]) {
    const T* x = (const T*)p.x + b * p.xb + c;
    long at[K - 1];
    int need = K - 1;                   // the oldest `need` are not found yet
#pragma unroll
    for (int k = 0; k < K - 1; ++k) at[k] = -1;
    if (!MASKED) {
        need = t0 < K - 1 ? (int)(K - 1 - t0) : 0;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) at[k] = t0 - (K - 1) + k;
    } else {
        const bool* mask = p.mask + b * p.steps;
        for (long end = t0; end > 0 && need > 0; end -= 64) {
            unsigned long long bits = seen_64(mask, end - 64, p.steps);
            if (bits && end < 64) bits &= ~0ull << (64 - end);
#pragma unroll
            for (int k = K - 2; k >= 0; --k) {
                if (k != need - 1 || !bits) continue;
                const int top = 63 - __clzll(bits);
                at[k] = end - 64 + top;
                bits ^= 1ull << top;
                --need;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        if (k >= need) {
            load_pack<T, V>(x + at[k] * p.xt, win[k]);
        } else if (p.state) {
            load_pack<T, V>((const T*)p.state + (b * (K - 1) + k + K - 1 - need) * p.width + c,
                            win[k]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) win[k][i] = 0.f;
        }
    }
}

// N floats that lie aligned, as wide as N allows.
template <int N> __device__ __forceinline__ void load_floats(const float* p, float* out) {
    constexpr int W = N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < N / W; ++i) load_pack<float, W>(p + i * W, out + i * W);
}

// The taps of a lane's channels: one run of memory, as a channel's K lie together.
template <int K, int V>
__device__ __forceinline__ void conv_weights(const ConvArgs& p, int c, float (&w)[K][V],
                                             float (&bias)[V]) {
    float run[K * V];
    load_floats<K * V>(p.w + (long)c * K, run);
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = run[i * K + k];
        bias[i] = 0.f;
    }
    if (p.bias) load_floats<V>(p.bias + c, bias);
}

constexpr int CU = 4;           // steps that a lane fetches at once

// A lane walks V channels of one tile of steps with the window in registers, so
// each input is read once but for the K-1 before each tile.  Memory bounds it:
// 4x4099x2048 bf16 takes 28 us on the GPU, 4.8 TB/s where a copy reaches 5.1.
template <typename T, int K, int V, bool MASKED>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvArgs p)
{
    const unsigned lanes = p.width / V;
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(at % lanes) * V;
    const long item = at / lanes;
    const long b = item / p.tiles;
    if (b >= p.batch) return;
    const long t0 = (item % p.tiles) * p.tile;
    const long t1 = t0 + p.tile < p.steps ? t0 + p.tile : p.steps;

    float w[K][V], bias[V], win[K - 1][V];
    const T* x = (const T*)p.x + b * p.xb + c;
    T* y = (T*)p.y + b * p.steps * p.width + c;
    const bool* mask = p.mask + b * p.steps;
    Pack<T, V> next[CU];
    int next_on[CU];            // a byte: turned into a bool here, it would be waited for
    auto fetch = [&](long t) {
#pragma unroll
        for (int u = 0; u < CU; ++u) {
            next_on[u] = t + u < t1;
            if (!next_on[u]) continue;
            next[u] = *(const Pack<T, V>*)(x + (t + u) * p.xt);
            if (MASKED) next_on[u] = ((const unsigned char*)mask)[t + u];
        }
    };
    fetch(t0);
    conv_weights<K, V>(p, c, w, bias);
    conv_behind<T, K, V, MASKED>(p, b, t0, c, win);
    for (long t = t0; t < t1; t += CU) {
        Pack<T, V> now[CU];
        int on[CU];
#pragma unroll
        for (int u = 0; u < CU; ++u) {
            now[u] = next[u];
            on[u] = next_on[u];
        }
        fetch(t + CU);
#pragma unroll
        for (int u = 0; u < CU; ++u) {
            if (t + u >= t1) break;
            float out[V] = {};
            if (on[u] & 1) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float v = to_float(now[u].v[i]);
                    float s = bias[i];
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) s = fmaf(w[k][i], win[k][i], s);
                    s = fmaf(w[K - 1][i], v, s);
                    out[i] = p.silu ? s * sigmoid(s) : s;
#pragma unroll
                    for (int k = 0; k < K - 2; ++k) win[k][i] = win[k + 1][i];
                    win[K - 2][i] = v;
                }
            }
            store_pack<T, V>(y + (t + u) * p.width, out);
        }
    }
    if (t1 == p.steps) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
            store_pack<T, V>((T*)p.last + (b * (K - 1) + k) * p.width + c, win[k]);
    }
}

// Backward: the lane walks its tile and K-1 observed steps behind it, so that
// every input of the tile has met all steps that used it.  Each input of the
// window has its gradient so far and its place: a step of the tile, none
// (another tile's), or one of the carried inputs.  128x16x512 takes 12 us, the
// time of 16 steps one behind the other, and the sum over its parts 4.
template <typename T, int K, int V, bool MASKED>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvArgs p)
{
    const unsigned lanes = p.width / V;
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(at % lanes) * V;
    const long part = at / lanes;
    if (part >= p.nparts) return;

    constexpr int none = -1, carried = -2;              // carried input j: -2 - j
    float w[K][V], bias[V], dw[K][V] = {}, db[V] = {};
    conv_weights<K, V>(p, c, w, bias);
    const long items = p.batch * p.tiles;
    for (long item = part; item < items; item += p.nparts) {
        const long b = item / p.tiles;
        const long t0 = (item % p.tiles) * p.tile;
        const long t1 = t0 + p.tile < p.steps ? t0 + p.tile : p.steps;
        const T* x = (const T*)p.x + b * p.xb + c;
        const T* dy = (const T*)p.dy + b * p.steps * p.width + c;
        T* dx = (T*)p.y + (b * p.steps + t0) * p.width + c;
        const bool* mask = p.mask + b * p.steps;

        float win[K - 1][V], acc[K - 1][V] = {};
        int place[K - 1];                               // steps from t0 on
        Pack<T, V> nx[CU], ng[CU];
        int non[CU];                                    // bytes, as a bool is waited for
        auto fetch = [&](long t) {
#pragma unroll
            for (int u = 0; u < CU; ++u) {
                non[u] = t + u < t1;
                if (!non[u]) continue;
                nx[u] = *(const Pack<T, V>*)(x + (t + u) * p.xt);
                ng[u] = *(const Pack<T, V>*)(dy + (t + u) * p.width);
                if (MASKED) non[u] = ((const unsigned char*)mask)[t + u];
            }
        };
        fetch(t0);
        conv_behind<T, K, V, MASKED>(p, b, t0, c, win);
        bool pending = false;                           // an input waits for more steps
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            place[k] = t0 == 0 ? carried - k : none;
            pending = pending || t0 == 0;
        }
        auto emit = [&](int to, const float (&g)[V]) {
            if (to >= 0)
                store_pack<T, V>(dx + (long)to * p.width, g);
            else if (to <= carried && p.last)
                store_pack<T, V>((T*)p.last + (b * (K - 1) + carried - to) * p.width + c, g);
        };
        // one observed step: its part in the taps and in the window's gradients
        auto step = [&](const Pack<T, V>& px, const Pack<T, V>& pg, int at) {
            float first[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float v = to_float(px.v[i]);
                float g = to_float(pg.v[i]);
                if (p.silu) {
                    float s = bias[i];
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) s = fmaf(w[k][i], win[k][i], s);
                    s = fmaf(w[K - 1][i], v, s);
                    const float sg = sigmoid(s);
                    g *= sg * (1.f + s * (1.f - sg));
                }
                if (at != none) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) dw[k][i] = fmaf(g, win[k][i], dw[k][i]);
                    dw[K - 1][i] = fmaf(g, v, dw[K - 1][i]);
                    db[i] += g;
                }
#pragma unroll
                for (int k = 0; k < K - 1; ++k) acc[k][i] = fmaf(w[k][i], g, acc[k][i]);
                first[i] = acc[0][i];
#pragma unroll
                for (int k = 0; k < K - 2; ++k) {
                    acc[k][i] = acc[k + 1][i];
                    win[k][i] = win[k + 1][i];
                }
                acc[K - 2][i] = w[K - 1][i] * g;
                win[K - 2][i] = v;
            }
            emit(place[0], first);
#pragma unroll
            for (int k = 0; k < K - 2; ++k) place[k] = place[k + 1];
            place[K - 2] = at;
        };
        for (long t = t0; t < t1; t += CU) {
            Pack<T, V> cx[CU], cg[CU];
            int on[CU];
#pragma unroll
            for (int u = 0; u < CU; ++u) {
                cx[u] = nx[u];
                cg[u] = ng[u];
                on[u] = non[u];
            }
            fetch(t + CU);
#pragma unroll
            for (int u = 0; u < CU; ++u) {
                if (t + u >= t1) break;
                if (on[u] & 1) {
                    step(cx[u], cg[u], (int)(t + u - t0));
                    pending = true;
                } else {
                    const float zero[V] = {};
                    store_pack<T, V>(dx + (t + u - t0) * p.width, zero);
                }
            }
        }
        // the K-1 observed steps behind the tile, where an input of it waits for them
        if (pending && t1 < p.steps) {
            long at[K - 1];
            int found = 0;
            if (!MASKED) {
                found = p.steps - t1 < K - 1 ? (int)(p.steps - t1) : K - 1;
#pragma unroll
                for (int k = 0; k < K - 1; ++k) at[k] = t1 + k;
            } else {
                for (long from = t1; from < p.steps && found < K - 1; from += 64) {
                    unsigned long long bits = seen_64(mask, from, p.steps);
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) {
                        if (k != found || !bits) continue;
                        at[k] = from + __builtin_ctzll(bits);
                        bits &= bits - 1;
                        ++found;
                    }
                }
            }
            Pack<T, V> ax[K - 1], ag[K - 1];
#pragma unroll
            for (int k = 0; k < K - 1; ++k) {
                if (k >= found) continue;
                ax[k] = *(const Pack<T, V>*)(x + at[k] * p.xt);
                ag[k] = *(const Pack<T, V>*)(dy + at[k] * p.width);
            }
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
                if (k < found) step(ax[k], ag[k], none);
        }
        // what the window still holds of this tile ended in the carried inputs
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            if (place[k] == none) continue;
            if (p.dlast) {
                float g[V];
                load_pack<T, V>((const T*)p.dlast + (b * (K - 1) + k) * p.width + c, g);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[k][i] += g[i];
            }
            emit(place[k], acc[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        store_pack<float, V>(p.parts + (part * (K + 1) + k) * p.width + c, dw[k]);
    store_pack<float, V>(p.parts + (part * (K + 1) + K) * p.width + c, db);
}

// One step of up to CU rows a lane, which then share its taps: 8192 x 512 bf16
// with every other row observed takes 8.3 us against 15.4 with a row a lane
// (33.6 MB; a copy of as much takes 6.6).
template <typename T, int K, int V>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvArgs p)
{
    const unsigned lanes = p.width / V;
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(at % lanes) * V;
    const long b0 = at / lanes * p.tile;
    if (b0 >= p.batch) return;
    Pack<T, V> win[CU][K];
    bool on[CU];
#pragma unroll
    for (int u = 0; u < CU; ++u) {
        const long b = b0 + u;
        on[u] = u < p.tile && b < p.batch && (!p.mask || p.mask[b]);
        if (!on[u]) continue;
        const T* state = (const T*)p.last + b * (K - 1) * p.width + c;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) win[u][k] = *(const Pack<T, V>*)(state + (long)k * p.width);
        win[u][K - 1] = *(const Pack<T, V>*)((const T*)p.x + b * p.xb + c);
    }
    float w[K][V], bias[V];
    conv_weights<K, V>(p, c, w, bias);
#pragma unroll
    for (int u = 0; u < CU; ++u) {
        const long b = b0 + u;
        if (u >= p.tile || b >= p.batch) break;
        float out[V] = {};
        if (on[u]) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s = bias[i];
#pragma unroll
                for (int k = 0; k < K; ++k) s = fmaf(w[k][i], to_float(win[u][k].v[i]), s);
                out[i] = p.silu ? s * sigmoid(s) : s;
            }
            T* state = (T*)p.last + b * (K - 1) * p.width + c;
#pragma unroll
            for (int k = 0; k < K - 1; ++k) *(Pack<T, V>*)(state + (long)k * p.width) = win[u][k + 1];
        }
        store_pack<T, V>((T*)p.y + b * p.width + c, out);
    }
}

// out[col] = sum over parts of parts[part][col], in a fixed order and 64 bits
// (up to 1024 parts of either sign).  Columns are (k, d); out is (d, k) for
// k < inner and goes to `rest` (d) for k == inner.
__global__ __launch_bounds__(256) void column_sum_kernel(
    const float* __restrict__ parts, long nparts, long width, int inner,
    float* __restrict__ out, float* __restrict__ rest)
{
    const long cols = width * (inner + (rest ? 1 : 0));
    const long col = (long)blockIdx.x * 16 + (threadIdx.x & 15);
    const int slice = threadIdx.x >> 4;
    double sum = 0;
    if (col < cols)
        for (long i = slice; i < nparts; i += 16) sum += parts[i * cols + col];
    __shared__ double s[16][17];
    s[slice][threadIdx.x & 15] = sum;
    __syncthreads();
    if (slice == 0 && col < cols) {
        for (int i = 1; i < 16; ++i) sum += s[i][threadIdx.x & 15];
        const long k = col / width, d = col % width;
        if (k < inner) out[d * inner + k] = (float)sum;
        else rest[d] = (float)sum;
    }
}

// ------------------------------------------------------------------- scan

struct ScanArgs {
    const void *x, *dt, *z, *B, *C;     // z may be null
    const float *A, *D, *bias;          // D, bias may be null
    const float* state;                 // (B, D, N) or null: zeros
    const bool* mask;                   // (B, T) or null
    const void* dy;                     // (B, T, D) dense
    const float* dlast;                 // (B, D, N) or null
    void* y;                            // (B, T, D) dense
    float* last;                        // (B, D, N)
    float* ckpt;                        // (B, chunks TC/TH, D, N) or null: h before each TH steps
    float *seg_h, *seg_d;               // (B, segs, D, N), (B, segs, D)
    void *dx, *ddt, *dz;                // (B, T, D)
    float *dBp, *dCp;                   // (tiles, B, T, G, N)
    float *dAp, *dDp;                   // (B segs, D, N), (B segs, 2, D): dD, dbias
    float* dstate;                      // (B, D, N) or null
    long batch, steps, chunks;
    long xb, xt, db, dt_, zb, zt, Bb, Bt, Bg, Cb, Ct, Cg;
    int width, states, per;
    unsigned groups, tiles, segs;
    int seg_chunks;
    int softplus, vec_d, vec_n, vec_b;
};

constexpr int TC = 16;          // steps of a chunk
constexpr int TH = 8;           // steps between the states that training keeps

// Sum over the L lanes of a channel; every lane gets it.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
        0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int L> __device__ __forceinline__ float channel_sum(float v) {
    if (L > 1) v += dpp<0xB1>(v);       // quad lanes 1 0 3 2
    if (L > 2) v += dpp<0x4E>(v);       // quad lanes 2 3 0 1
    if (L > 4) v += dpp<0x141>(v);      // the half row backwards
    if (L > 8) v += dpp<0x140>(v);      // the row backwards
    return v;
}

// Adds a to b across the halves of a wave (32) or across neighbouring rows of
// 16 lanes (16): the first lanes of each pair get a's sum, the others b's.
__device__ __forceinline__ float fold32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(
        __builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned lo = r[0], hi = r[1];    // a bit_cast of r[1] itself reads r[0]
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float fold16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(
        __builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned lo = r[0], hi = r[1];
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// Sums eight values over a wave's channels (lanes L apart), halving the number
// of values with each exchange: 16 instructions for L = 4 instead of 8 x 4
// exchanges and sums.  The sum of vb[i] is then in the lanes with bit 5 of i's
// bit 0 and bit 4 of its bit 1, that of vc[i] in those with bit 3 set too (for
// L = 16: in the second value).
template <int L>
__device__ __forceinline__ void wave_fold(const float (&vb)[4], const float (&vc)[4],
                                          float& first, float& second) {
    const float b = fold16(fold32(vb[0], vb[1]), fold32(vb[2], vb[3]));
    const float c = fold16(fold32(vc[0], vc[1]), fold32(vc[2], vc[3]));
    if (L == 16) {
        first = b;
        second = c;
        return;
    }
    const bool upper = threadIdx.x & 8;
    float v = upper ? c : b, w = upper ? b : c;
    v += dpp<0x128>(w);                 // the row turned by 8
    if (L < 8) v += dpp<0x104>(v);      // from 4 lanes above
    if (L < 4) v += dpp<0x4E>(v);
    if (L < 2) v += dpp<0xB1>(v);
    first = second = v;
}

// Which rows, channels and steps a block has: 256 threads take 256/L channels
// of one group, L lanes a channel and four states a lane.
template <int L> struct Place {
    static constexpr int CB = 256 / L;
    long b;
    int g, seg, tile, c0, nc;           // first channel, how many
    int c, n0, nn;                      // this lane's channel in the block, its states
    bool live;
    __device__ __forceinline__ Place(const ScanArgs& p) {
        unsigned at = blockIdx.x;
        tile = at % p.tiles; at /= p.tiles;
        g = at % p.groups; at /= p.groups;
        seg = at % p.segs;
        b = at / p.segs;
        c0 = g * p.per + tile * CB;
        nc = min(CB, p.per - tile * CB);
        c = threadIdx.x / L;
        n0 = 4 * (threadIdx.x % L);
        live = c < nc;
        nn = live ? min(4, max(0, p.states - n0)) : 0;
    }
    __device__ __forceinline__ long state_at(const ScanArgs& p, long row) const {
        return (row * p.width + c0 + c) * p.states + n0;
    }
};

// A thread's part of a chunk's values: four channels of a step at a time.
template <int L> struct Part {
    static constexpr int groups = TC * (256 / L) / 4;
    static constexpr int count = (groups + 255) / 256;
    int t, c;
    bool in;                            // the part exists
    __device__ __forceinline__ Part(int k) {
        const int at = threadIdx.x + 256 * k;
        in = at < groups;
        t = at / (256 / L / 4);
        c = 4 * (at % (256 / L / 4));
    }
};

// What a thread reads of a chunk, as it lies in memory: fetched while the chunk
// before is computed.  Of unobserved steps it may hold anything; `on` tells.
template <typename T, int L> struct Chunk {
    static constexpr int NQ = Part<L>::count;
    Pack<T, 4> x[NQ], dt[NQ], z[NQ], dy[NQ], B, C;
    bool on[NQ], on_bc;

    template <bool X, bool Z, bool DY, bool HAS_B, bool HAS_C>
    __device__ __forceinline__ void fetch(const ScanArgs& p, const Place<L>& at, long t0) {
        const bool* mask = p.mask ? p.mask + at.b * p.steps : nullptr;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const Part<L> q(j);
            const long s = t0 + q.t;
            const int n = at.nc - q.c, c = at.c0 + q.c;
            on[j] = q.in && n > 0 && s < p.steps;
            if (!on[j]) continue;
            if (X) x[j] = load_raw((const T*)p.x + at.b * p.xb + s * p.xt + c, n, p.vec_d);
            dt[j] = load_raw((const T*)p.dt + at.b * p.db + s * p.dt_ + c, n, p.vec_d);
            if (Z && p.z) z[j] = load_raw((const T*)p.z + at.b * p.zb + s * p.zt + c, n, p.vec_d);
            if (DY)
                dy[j] = load_raw((const T*)p.dy + (at.b * p.steps + s) * p.width + c, n, p.vec_d);
            if (mask) on[j] = mask[s];
        }
        const int t = threadIdx.x / L, n = 4 * (threadIdx.x % L);
        const long s = t0 + t;
        on_bc = t < TC && s < p.steps && n < p.states;
        if (on_bc) {
            if (HAS_B)
                B = load_raw((const T*)p.B + at.b * p.Bb + s * p.Bt + at.g * p.Bg + n,
                             p.states - n, p.vec_b);
            if (HAS_C)
                C = load_raw((const T*)p.C + at.b * p.Cb + s * p.Ct + at.g * p.Cg + n,
                             p.states - n, p.vec_b);
            if (mask) on_bc = mask[s];
        }
    }

    template <bool HAS_B, bool HAS_C>
    __device__ __forceinline__ void stage_bc(float (*sB)[4 * L], float (*sC)[4 * L]) const {
        const int t = threadIdx.x / L, n = 4 * (threadIdx.x % L);
        if (t >= TC) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (HAS_B) sB[t][n + i] = on_bc ? to_float(B.v[i]) : 0.f;
            if (HAS_C) sC[t][n + i] = on_bc ? to_float(C.v[i]) : 0.f;
        }
    }
};

// A rate times log2(e).  One past a float's range, an infinite one among them, stays
// at its end: a step of length 0, unobserved or behind the last, has to take 0 * rate.
__device__ __forceinline__ float rate_of(float a) {
    const float r = a * kLog2e, most = __FLT_MAX__;
    return r > most ? most : r < -most ? -most : r;     // NaN stays
}

// A lane's rates.
template <int L>
__device__ __forceinline__ void load_rates(const ScanArgs& p, const Place<L>& at, float* A2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] = 0.f;
    if (at.nn > 0) load4(p.A + (long)(at.c0 + at.c) * p.states + at.n0, at.nn, p.vec_n, A2);
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] = rate_of(A2[i]);
}

// A thread's four values of D or dt_bias; zeros where there are none.
template <int L>
__device__ __forceinline__ void load_channels(const float* from, const Place<L>& at, float* out) {
    const Part<L> q(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = from && q.c + i < at.nc ? from[at.c0 + q.c + i] : 0.f;
}

// h e^(ln2 p).  A whole segment's factor may pass the range of a float where its
// product with a small state, or one of 0, does not, so p's whole part goes to the
// exponent of the product; behind 600 the product of any float but 0 has left the
// range.  A p that is not a number comes back in `e` below.  This costs 4 of the
// 114 us that the walk of 4x2048x2048 takes, 1.5 of 68 for 1x8192x1024.
__device__ __forceinline__ float grown(float h, float p) {
    p = fminf(fmaxf(p, -600.f), 600.f);
    const float whole = rintf(p);
    return ldexpf(exp2_fast(p - whole) * h, (int)whole);
}

// Moves a state (or, backwards, the gradient of one) through whole segments.
template <int L>
__device__ __forceinline__ void join_segment(const ScanArgs& p, const Place<L>& at, int seg,
                                             const float* A2, float* h) {
    const long row = at.b * p.segs + seg;
    float e[4];
    load4(p.seg_h + at.state_at(p, row), at.nn, p.vec_n, e);
    const float d = p.seg_d[row * p.width + at.c0 + at.c];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = grown(h[i], A2[i] * d) + e[i];
}

// What a lane reads of one step.  The next step's is read before the present one
// is computed: the compiler alone reads just before the use, and each step then
// waits for shared memory (4x2048x2048 backward: 347 us against 318).
struct StepIn {
    float2 v;
    float g, B[4], C[4];
    template <bool HAS_G, bool HAS_B, bool HAS_C>
    __device__ __forceinline__ void read(const float2* sv, const float* sg, const float* sB,
                                         const float* sC, int c, int n0) {
        v = sv[c];
        if (HAS_G) g = sg[c];
        if (HAS_B) load_pack<float, 4>(sB + n0, B);
        if (HAS_C) load_pack<float, 4>(sC + n0, C);
    }
};

// LOCAL: the segment's own end from a zero start, and its sum of d, for the
// segments behind it.  Otherwise the outputs, from the state before the
// segment: the carried one moved through the segments before.  Vector
// instructions bound both: 17 and 23 a step of four states, and 0.3 as many to
// stage a chunk.  4x2048x2048 with 16 states, 8 segments: 65 and 114 us (of the
// memory's rate they take 0.5 and 2.5 TB/s).
template <typename T, int L, bool LOCAL>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanArgs p)
{
    const Place<L> at(p);
    if (LOCAL && at.seg == (int)p.segs - 1) return;     // nothing lies behind it
    constexpr int NQ = Part<L>::count;
    __shared__ __attribute__((aligned(16))) float2 sdu[TC][256 / L];
    __shared__ __attribute__((aligned(16))) float sB[TC][4 * L], sC[TC][4 * L], sy[TC][256 / L];

    float A2[4], h[4] = {}, total = 0.f, Dv[4], bias[4];
    load_rates<L>(p, at, A2);
    load_channels<L>(p.bias, at, bias);
    if (!LOCAL) {
        load_channels<L>(p.D, at, Dv);
        if (at.nn > 0) {
            if (p.state) load4(p.state + at.state_at(p, at.b), at.nn, p.vec_n, h);
            for (int s = 0; s < at.seg; ++s) join_segment<L>(p, at, s, A2, h);
        }
    }
    const long k0 = (long)at.seg * p.seg_chunks;
    const long k1 = min(k0 + p.seg_chunks, p.chunks);
    Chunk<T, L> next;
    next.template fetch<true, !LOCAL, false, true, !LOCAL>(p, at, k0 * TC);
    for (long k = k0; k < k1; ++k) {
        const long t0 = k * TC;
        const Chunk<T, L> now = next;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const Part<L> q(j);
            if (!q.in) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float raw = to_float(now.dt[j].v[i]) + bias[i];
                const float d = now.on[j] ? (p.softplus ? softplus(raw) : raw) : 0.f;
                const float x = now.on[j] ? to_float(now.x[j].v[i]) : 0.f;
                sdu[q.t][q.c + i] = make_float2(d, d * x);
            }
        }
        now.template stage_bc<true, !LOCAL>(sB, sC);
        __syncthreads();
        if (k + 1 < k1) next.template fetch<true, !LOCAL, false, true, !LOCAL>(p, at, t0 + TC);
        // steps behind the end have d = 0 and x = 0 and change nothing
        StepIn in[2];
        in[0].template read<false, true, !LOCAL>(sdu[0], nullptr, sB[0], sC[0], at.c, at.n0);
#pragma unroll
        for (int t = 0; t < TC; ++t) {
            if (!LOCAL && t % TH == 0 && p.ckpt && at.nn > 0)
                store4(p.ckpt + at.state_at(p, (at.b * p.chunks + k) * (TC / TH) + t / TH), at.nn,
                       p.vec_n, h);
            if (t + 1 < TC)
                in[(t + 1) & 1].template read<false, true, !LOCAL>(
                    sdu[t + 1], nullptr, sB[t + 1], sC[t + 1], at.c, at.n0);
            const StepIn& s = in[t & 1];
            float y = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = fmaf(exp2_fast(A2[i] * s.v.x), h[i], s.v.y * s.B[i]);
                if (!LOCAL) y = fmaf(s.C[i], h[i], y);
            }
            if (LOCAL) total += s.v.x;
            else sy[t][at.c] = channel_sum<L>(y);       // the same from all its lanes
        }
        __syncthreads();
        if (LOCAL) continue;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const Part<L> q(j);
            const long s = t0 + q.t;
            if (!q.in || q.c >= at.nc || s >= p.steps) continue;
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                y[i] = fmaf(Dv[i], to_float(now.x[j].v[i]), sy[q.t][q.c + i]);
                if (p.z) {
                    const float z = to_float(now.z[j].v[i]);
                    y[i] *= z * sigmoid(z);
                }
                if (!now.on[j]) y[i] = 0.f;
            }
            store4((T*)p.y + (at.b * p.steps + s) * p.width + at.c0 + q.c, at.nc - q.c, p.vec_d, y);
        }
    }
    if (LOCAL) {
        const long row = at.b * p.segs + at.seg;
        if (at.nn > 0) store4(p.seg_h + at.state_at(p, row), at.nn, p.vec_n, h);
        if (at.live && at.n0 == 0) p.seg_d[row * p.width + at.c0 + at.c] = total;
    } else if (at.seg == (int)p.segs - 1 && at.nn > 0) {
        store4(p.last + at.state_at(p, at.b), at.nn, p.vec_n, h);
    }
}

// Backward.  With g_t the gradient of C.h + D x and lam_t that of h_t:
//   lam_t = C_t g_t + carry,  carry <- exp(d_t A) lam_t
// LOCAL: a segment's carry from a zero one behind it.  Otherwise the
// gradients: h is walked again from a kept state and stays in registers with
// exp(d A), then the same steps are walked backwards.  4x2048x2048 with 16
// states, 8 segments: 74 and 327 us; of the latter's issue slots vector
// instructions take 65 to 70 %, a fifth of them to stage and to store a chunk.
// Eight steps of states and decays at a time stay below 256 registers: 593 us
// for training 4x2048x2048 against 633 with sixteen, which spill.
template <typename T, int L, bool LOCAL>
__global__ __launch_bounds__(256, LOCAL ? 4 : 2) void scan_bwd_kernel(ScanArgs p)
{
    constexpr int CB = 256 / L, NP = 4 * L, CW = 64 / L, NQ = Part<L>::count;
    const Place<L> at(p);
    if (LOCAL && at.seg == 0) return;                   // nothing lies before it
    __shared__ __attribute__((aligned(16))) float2 sdx[TC][CB];     // d, x
    __shared__ __attribute__((aligned(16))) float sg[TC][CB], sB[TC][NP], sC[TC][NP];
    // each wave's sums lam B and A2 a h lam of its channels, C h, and its dB and dC
    __shared__ float ss[LOCAL ? 1 : TC][4][2][CW], sy[LOCAL ? 1 : TC][CB];
    __shared__ float sbc[LOCAL ? 1 : 4][TC + 1][2][NP];             // the last row for none

    float A2[4], lam[4] = {}, dA[4] = {}, total = 0.f, bias[4], Dv[4];
    float dD[4] = {}, dbias[4] = {}, first[4] = {};
    load_rates<L>(p, at, A2);
    load_channels<L>(p.bias, at, bias);
    if (!LOCAL) {
        load_channels<L>(p.D, at, Dv);
        if (at.nn > 0) {
            if (p.dlast) load4(p.dlast + at.state_at(p, at.b), at.nn, p.vec_n, lam);
            for (int s = (int)p.segs - 1; s > at.seg; --s) join_segment<L>(p, at, s, A2, lam);
        }
    }
    const long k0 = (long)at.seg * p.seg_chunks;
    const long k1 = min(k0 + p.seg_chunks, p.chunks);
    Chunk<T, L> next;
    next.template fetch<!LOCAL, true, true, !LOCAL, true>(p, at, (k1 - 1) * TC);
    if (!LOCAL && at.nn > 0)
        load4(p.ckpt + at.state_at(p, (at.b * p.chunks + k1) * (TC / TH) - 1), at.nn, p.vec_n, first);
    for (long k = k1 - 1; k >= k0; --k) {
        const long t0 = k * TC;
        const Chunk<T, L> now = next;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const Part<L> q(j);
            if (!q.in) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float raw = to_float(now.dt[j].v[i]) + bias[i];
                const float d = now.on[j] ? (p.softplus ? softplus(raw) : raw) : 0.f;
                float g = to_float(now.dy[j].v[i]);
                if (p.z) {
                    const float z = to_float(now.z[j].v[i]);
                    g *= z * sigmoid(z);
                }
                sdx[q.t][q.c + i] = make_float2(d, !LOCAL && now.on[j] ? to_float(now.x[j].v[i]) : 0.f);
                sg[q.t][q.c + i] = now.on[j] ? g : 0.f;
            }
        }
        now.template stage_bc<!LOCAL, true>(sB, sC);
        __syncthreads();
        if (k > k0) next.template fetch<!LOCAL, true, true, !LOCAL, true>(p, at, t0 - TC);

        if (LOCAL) {
            StepIn in[2];
            in[1].template read<true, false, true>(sdx[TC - 1], sg[TC - 1], nullptr, sC[TC - 1],
                                                   at.c, at.n0);
#pragma unroll
            for (int t = TC - 1; t >= 0; --t) {
                if (t > 0)
                    in[(t - 1) & 1].template read<true, false, true>(sdx[t - 1], sg[t - 1], nullptr,
                                                                     sC[t - 1], at.c, at.n0);
                const StepIn& s = in[t & 1];
                total += s.v.x;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    lam[i] = exp2_fast(A2[i] * s.v.x) * fmaf(s.C[i], s.g, lam[i]);
            }
            __syncthreads();
            continue;
        } else {
            // where a lane's share of the sums goes
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            const bool has = L == 16 || (lane & 7) < L;
            float* to_bc = &sbc[wave][has ? 0 : TC][L < 16 ? (lane >> 3) & 1 : 0]
                               [at.n0 + (lane >> 5) + 2 * ((lane >> 4) & 1)];
            const int step_bc = has ? 2 * NP : 0;
            float* to_s = &ss[0][wave][L > 1 && (at.n0 & 4) ? 1 : 0][lane / L];
#pragma unroll 1
            for (int u = TC - TH; u >= 0; u -= TH) {
                float hs[TH + 1][4], a[TH][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) hs[0][i] = first[i];
                const long row = (at.b * p.chunks + k) * (TC / TH) + u / TH - 1;
                if ((k > k0 || u > 0) && at.nn > 0)
                    load4(p.ckpt + at.state_at(p, row), at.nn, p.vec_n, first);
                StepIn in[2];
                in[0].template read<false, true, true>(sdx[u], nullptr, sB[u], sC[u], at.c, at.n0);
#pragma unroll
                for (int t = 0; t < TH; ++t) {
                    if (t + 1 < TH)
                        in[(t + 1) & 1].template read<false, true, true>(
                            sdx[u + t + 1], nullptr, sB[u + t + 1], sC[u + t + 1], at.c, at.n0);
                    else
                        in[t & 1].g = sg[u + t][at.c];  // where the way back begins
                    const StepIn& s = in[t & 1];
                    const float du = s.v.x * s.v.y;
                    float y = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        a[t][i] = exp2_fast(A2[i] * s.v.x);
                        hs[t + 1][i] = fmaf(a[t][i], hs[t][i], du * s.B[i]);
                        y = fmaf(s.C[i], hs[t + 1][i], y);
                    }
                    sy[u + t][at.c] = channel_sum<L>(y);        // the same from all its lanes
                }
#pragma unroll
                for (int t = TH - 1; t >= 0; --t) {
                    if (t > 0)
                        in[(t - 1) & 1].template read<true, true, true>(
                            sdx[u + t - 1], sg[u + t - 1], sB[u + t - 1], sC[u + t - 1], at.c, at.n0);
                    const StepIn& s = in[t & 1];
                    const float du = s.v.x * s.v.y;
                    float s1 = 0.f, s2 = 0.f, vb[4], vc[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float l = fmaf(s.C[i], s.g, lam[i]);
                        vc[i] = s.g * hs[t + 1][i];
                        vb[i] = l * du;
                        s1 = fmaf(l, s.B[i], s1);
                        lam[i] = a[t][i] * l;
                        const float ah = lam[i] * hs[t][i];
                        s2 = fmaf(A2[i], ah, s2);
                        dA[i] = fmaf(s.v.x, ah, dA[i]);
                    }
                    s1 = channel_sum<L>(s1);
                    s2 = channel_sum<L>(s2);
                    if (L > 1) {
                        to_s[(u + t) * 8 * CW] = (at.n0 & 4) ? s2 : s1;
                    } else {
                        to_s[(u + t) * 8 * CW] = s1;
                        to_s[(u + t) * 8 * CW + CW] = s2;
                    }
                    float b, c;
                    wave_fold<L>(vb, vc, b, c);
                    to_bc[(u + t) * step_bc] = b;
                    if (L == 16) to_bc[(u + t) * step_bc + NP] = c;
                }
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                const Part<L> q(j);
                const long s = t0 + q.t;
                if (!q.in || q.c >= at.nc || s >= p.steps) continue;
                const int n = at.nc - q.c;
                float dx[4], dd[4], dz[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int w = (q.c + i) / CW, cw = (q.c + i) % CW;
                    const float s1 = ss[q.t][w][0][cw], s2 = ss[q.t][w][1][cw];
                    const float g = sg[q.t][q.c + i];
                    const float2 v = sdx[q.t][q.c + i];         // d and x, 0 where unobserved
                    dx[i] = fmaf(v.x, s1, Dv[i] * g);
                    dd[i] = fmaf(v.y, s1, kLn2 * s2);
                    if (p.softplus) dd[i] *= sigmoid(to_float(now.dt[j].v[i]) + bias[i]);
                    if (!now.on[j]) dd[i] = 0.f;
                    dD[i] = fmaf(g, v.y, dD[i]);
                    dbias[i] += dd[i];
                    if (p.z) {
                        const float z = to_float(now.z[j].v[i]), sz = sigmoid(z);
                        dz[i] = to_float(now.dy[j].v[i]) * fmaf(Dv[i], v.y, sy[q.t][q.c + i]) *
                                sz * (1.f + z * (1.f - sz));
                        if (!now.on[j]) dz[i] = 0.f;
                    }
                }
                const long to = (at.b * p.steps + s) * p.width + at.c0 + q.c;
                store4((T*)p.dx + to, n, p.vec_d, dx);
                store4((T*)p.ddt + to, n, p.vec_d, dd);
                if (p.z) store4((T*)p.dz + to, n, p.vec_d, dz);
            }
            for (int e = threadIdx.x; e < TC * NP; e += 256) {
                const int t = e / NP, n = e % NP;
                const long s = t0 + t;
                if (n >= p.states || s >= p.steps) continue;
                const long to = (((at.tile * p.batch + at.b) * p.steps + s) * p.groups + at.g) *
                                p.states + n;
                float vb = 0.f, vc = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    vb += sbc[w][t][0][n];
                    vc += sbc[w][t][1][n];
                }
                p.dBp[to] = vb;
                p.dCp[to] = vc;
            }
            __syncthreads();
        }
    }
    const long row = at.b * p.segs + at.seg;
    if (LOCAL) {
        if (at.nn > 0) store4(p.seg_h + at.state_at(p, row), at.nn, p.vec_n, lam);
        if (at.live && at.n0 == 0) p.seg_d[row * p.width + at.c0 + at.c] = total;
    } else {
        if (at.seg == 0 && p.dstate && at.nn > 0)
            store4(p.dstate + at.state_at(p, at.b), at.nn, p.vec_n, lam);
        if (at.nn > 0) store4(p.dAp + at.state_at(p, row), at.nn, p.vec_n, dA);
        // dD and dbias: a thread has its four channels over its steps of each chunk
        float* fold = (float*)sdx;
        constexpr int rows = 256 / (CB / 4);
        const int c4 = 4 * (threadIdx.x % (CB / 4)), r = threadIdx.x / (CB / 4);
        for (int which = 0; which < 2; ++which) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r < TC) fold[r * CB + c4 + i] = which ? dbias[i] : dD[i];
            __syncthreads();
            for (int c = threadIdx.x; c < at.nc; c += 256) {
                float s = 0.f;
                for (int i = 0; i < (rows < TC ? rows : TC); ++i) s += fold[i * CB + c];
                p.dDp[(row * 2 + which) * p.width + at.c0 + c] = s;
            }
            __syncthreads();
        }
    }
}

// The rest of the backward pass in one launch, each block one part of it: sums
// dB and dC over the channel tiles (and rounds them once), and dA, dD and dbias
// over rows and segments, in a fixed order and 64 bits.  `first` is the launch's
// first part, where one launch cannot hold them all.
template <typename T>
__global__ __launch_bounds__(256) void scan_finish_kernel(
    const float* __restrict__ bc, int tiles, long nbc, T* __restrict__ dB, T* __restrict__ dC,
    const float* __restrict__ dAp, const float* __restrict__ dDp, long rows, long nA, long nD,
    float* __restrict__ dA, float* __restrict__ dD, long first)
{
    __shared__ double fold[16][17];
    const long blocks_bc = (nbc + 255) / 256;
    long at = first + blockIdx.x;
    if (at < 2 * blocks_bc) {
        const bool second = at >= blocks_bc;
        const long i = (second ? at - blocks_bc : at) * 256 + threadIdx.x;
        if (i >= nbc) return;
        const float* from = bc + (second ? tiles * nbc : 0) + i;
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < tiles; ++k) s += from[k * nbc];
        (second ? dC : dB)[i] = from_float<T>(s);
        return;
    }
    at -= 2 * blocks_bc;
    const long blocks_A = (nA + 15) / 16;
    const bool second = at >= blocks_A;
    const long cols = second ? nD : nA;
    const long col = (second ? at - blocks_A : at) * 16 + (threadIdx.x & 15);
    const float* from = second ? dDp : dAp;
    const int slice = threadIdx.x >> 4;
    double sum = 0;
    if (col < cols) {
#pragma unroll 4
        for (long i = slice; i < rows; i += 16) sum += from[i * cols + col];
    }
    fold[slice][threadIdx.x & 15] = sum;
    __syncthreads();
    if (slice == 0 && col < cols) {
        for (int i = 1; i < 16; ++i) sum += fold[i][threadIdx.x & 15];
        (second ? dD : dA)[col] = (float)sum;
    }
}

struct StepArgs {
    const void *x, *dt, *z, *B, *C;
    const float *A, *D, *bias;
    const bool* mask;
    float* state;
    void* y;
    long batch, xb, db, zb, Bb, Bg, Cb, Cg;
    int width, states, groups, per, rows, softplus, vec_n, vec_b;
};

// A state's four values, past the caches where `once` says that they are far
// more than those hold.
typedef float float4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Pack<float, 4> load_once(const float* p, int n, bool whole, bool once) {
    if (!whole || !once) return load_raw(p, n, whole);
    return __builtin_bit_cast(Pack<float, 4>, __builtin_nontemporal_load((const float4v*)p));
}
__device__ __forceinline__ void store_once(float* p, int n, bool whole, bool once,
                                           const Pack<float, 4>& h) {
    if (whole && once) __builtin_nontemporal_store(__builtin_bit_cast(float4v, h), (float4v*)p);
    else store4(p, n, whole, h.v);
}

constexpr int SR = 2;           // rows that a lane of a large step has in flight

// One step: four states a lane, L lanes a channel, the state in place.  What
// bounds it is the state's way to the lane and back.  8192 x 512 x 16 with every
// other row observed (286 MB): 114 us with a row a lane, 102 with two, 85 with
// the masks read first and the state past the caches (105 with one row; these as
// replayed graphs: a launch among others takes the last 79); four rows a lane
// take 91, for their registers take waves.
template <typename T, int L>
__global__ __launch_bounds__(256) void scan_step_kernel(StepArgs p)
{
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    const int n0 = 4 * (int)(at % L);
    const long item = at / L;                           // (rows, channel)
    const unsigned width = p.width;
    const long b0 = item / width * p.rows;
    const int c = (int)(item % width), g = c / p.per;
    const int have = min(4, p.states - n0);             // none of a lane behind the states
    Pack<float, 4> h[SR];
    Pack<T, 4> vb[SR], vc[SR];
    T x[SR], dt[SR], z[SR];
    float A[4] = {};
    bool in[SR], on[SR];
#pragma unroll
    for (int u = 0; u < SR; ++u) {
        in[u] = u < p.rows && b0 + u < p.batch;
        on[u] = in[u];
        if (in[u] && p.mask) on[u] = p.mask[b0 + u];
    }
#pragma unroll
    for (int u = 0; u < SR; ++u) {
        const long b = b0 + u;
        if (!on[u]) continue;
        if (have > 0) {
            h[u] = load_once(p.state + (b * width + c) * p.states + n0, have, p.vec_n, p.rows > 1);
            vb[u] = load_raw((const T*)p.B + b * p.Bb + g * p.Bg + n0, have, p.vec_b);
            vc[u] = load_raw((const T*)p.C + b * p.Cb + g * p.Cg + n0, have, p.vec_b);
        }
        x[u] = ((const T*)p.x)[b * p.xb + c];
        dt[u] = ((const T*)p.dt)[b * p.db + c];
        if (p.z) z[u] = ((const T*)p.z)[b * p.zb + c];
    }
    if (have > 0) load4(p.A + (long)c * p.states + n0, have, p.vec_n, A);
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] *= kLog2e;
    const float bias = p.bias ? p.bias[c] : 0.f, D = p.D ? p.D[c] : 0.f;
#pragma unroll
    for (int u = 0; u < SR; ++u) {
        const long row = (b0 + u) * width + c;
        float y = 0.f;
        if (on[u] && have > 0) {
            const float raw = to_float(dt[u]) + bias;
            const float d = p.softplus ? softplus(raw) : raw, du = d * to_float(x[u]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[u].v[i] = fmaf(exp2_fast(A[i] * d), h[u].v[i], du * to_float(vb[u].v[i]));
                y = fmaf(to_float(vc[u].v[i]), h[u].v[i], y);
            }
            store_once(p.state + row * p.states + n0, have, p.vec_n, p.rows > 1, h[u]);
        }
        y = channel_sum<L>(y);
        if (in[u] && n0 == 0) {
            if (on[u]) {
                y = fmaf(D, to_float(x[u]), y);
                if (p.z) y *= to_float(z[u]) * sigmoid(to_float(z[u]));
            }
            ((T*)p.y)[row] = from_float<T>(on[u] ? y : 0.f);
        }
    }
}

// ------------------------------------------------------------------- host

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// The kernels read the last axis dense; anything else is laid out anew.
Tensor dense_last(const Tensor& t) {
    return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

bool aligned(const Tensor& t, int v) {
    if ((uintptr_t)t.data_ptr() % (v * t.element_size())) return false;
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) % v) return false;
    return true;
}

void check_like(const char* op, const char* name, const Tensor& t, const Tensor& x,
                torch::ScalarType type, at::IntArrayRef shape)
{
    TORCH_CHECK_VALUE(t.device() == x.device(), op, ": ", name, " is on ", t.device(),
                      ", x on ", x.device());
    TORCH_CHECK_VALUE(t.scalar_type() == type, op, ": ", name, " must be ", type, ", got ",
                      t.scalar_type());
    TORCH_CHECK_VALUE(t.sizes() == shape, op, ": ", name, " must have shape ", shape, ", got ",
                      t.sizes());
}

void check_x(const char* op, const Tensor& x, int64_t dim)
{
    TORCH_CHECK_VALUE(x.is_cuda(), op, ": x must be on the GPU");
    TORCH_CHECK_VALUE(x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16,
                      op, ": x must be float32 or bfloat16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() == dim && x.size(-1) >= 1, op, ": x must be ",
                      dim == 3 ? "(batch, steps, channels)" : "(batch, channels)", ", got ",
                      x.sizes());
    TORCH_CHECK_VALUE(x.size(-1) < (1L << 24), op, ": too many channels");
}

// (B, T), or (B, T, 1), of truth values or numbers: 0 is unobserved.
Tensor as_mask(const char* op, const OptTensor& mask, const Tensor& x)
{
    if (!mask) return Tensor();
    auto want = x.sizes().slice(0, x.dim() - 1);
    auto m = *mask;
    if (m.dim() == x.dim() && m.size(-1) == 1) m = m.squeeze(-1);
    TORCH_CHECK_VALUE(m.device() == x.device(), op, ": mask is on ", m.device(), ", x on ",
                      x.device());
    TORCH_CHECK_VALUE(m.sizes() == want, op, ": mask must have shape ", want, ", got ",
                      mask->sizes());
    return (m.scalar_type() == torch::kBool ? m : m.ne(0)).contiguous();
}

// A launch counts its threads in 32 bits.
constexpr int64_t kMostBlocks = (1LL << 24) - 1;

int64_t blocks_for(int64_t threads, const char* op)
{
    const int64_t n = (threads + 255) / 256;
    TORCH_CHECK_VALUE(n <= kMostBlocks, op, ": too large for one launch, share out the batch");
    return n;
}

template <typename F> void by_type(const Tensor& x, F f)
{
    if (x.scalar_type() == torch::kBFloat16) f(bf16());
    else f(float());
}
template <int N> struct Const { static constexpr int value = N; };

// A step changes the state behind torch's back: tell autograd's version check.
void moved_on(const Tensor& state) {
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
}

// ---- convolution

template <typename F> void by_taps(int64_t taps, F f)
{
    if (taps == 2) f(Const<2>());
    else if (taps == 3) f(Const<3>());
    else f(Const<4>());
}

template <typename F> void by_conv(const Tensor& x, int64_t taps, int channels, F f)
{
    by_type(x, [&](auto t) {
        by_taps(taps, [&](auto k) {
            if (channels == 2) f(t, k, Const<2>());
            else f(t, k, Const<1>());
        });
    });
}

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const float* fptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const bool* mptr(const Tensor& t) { return t.defined() ? t.data_ptr<bool>() : nullptr; }

ConvArgs conv_args(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state,
                   const Tensor& mask, bool silu)
{
    ConvArgs p{};
    p.x = ptr(x); p.w = fptr(w); p.bias = fptr(bias); p.state = ptr(state); p.mask = mptr(mask);
    p.batch = x.size(0); p.steps = x.dim() == 3 ? x.size(1) : 1;
    p.xb = x.stride(0); p.xt = x.dim() == 3 ? x.stride(1) : 0;
    p.width = (int)x.size(-1); p.silu = silu;
    return p;
}

// Channels that a lane takes: two where all the tensors allow it.  More of them
// (16 bytes) made 4x4099x2048 bf16 slower, 32 us against 27, for they take the
// registers of waves that would hide the loads.
int conv_channels(const Tensor& x, std::initializer_list<Tensor> others)
{
    bool ok = x.size(-1) % 2 == 0 && aligned(x, 2);
    for (auto& t : others) ok = ok && (!t.defined() || aligned(t, 2));
    return ok ? 2 : 1;
}

// Steps of a lane's tile: 64, or down to 16 where that leaves fewer than 2^18
// lanes.  With gaps, fp32 1x7178x902: 26 us at 64 steps, 21 at 32, 20 at 16; with
// lanes enough, bf16 6x2735x975: 41 us at 64 and 32, 46 at 16, where the walk for
// the observed steps behind weighs more.  4x4099x2048: 28 us at 64 as at 32.
void cut_conv(ConvArgs& p, int channels)
{
    for (p.tile = 64; p.tile > 16; p.tile /= 2)
        if (p.batch * (p.width / channels) * ((p.steps + p.tile - 1) / p.tile) >= 1 << 18) break;
    p.tiles = (int)((p.steps + p.tile - 1) / p.tile);
}

std::vector<Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias,
                                 const Tensor& state, const Tensor& mask, bool silu)
{
    const c10::DeviceGuard guard(x.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    const int64_t taps = w.size(1);
    ConvArgs p = conv_args(x, w, bias, state, mask, silu);
    const int channels = conv_channels(x, {state});
    cut_conv(p, channels);
    const int64_t n = blocks_for(p.batch * p.tiles * (p.width / channels), "causal_conv");
    auto y = torch::empty(x.sizes(), x.options());
    auto last = torch::empty({x.size(0), taps - 1, x.size(2)}, x.options());
    if (p.batch == 0 || p.steps == 0) {
        if (state.defined()) last.copy_(state); else last.zero_();
        return {y, last};
    }
    p.y = y.data_ptr(); p.last = last.data_ptr();
    by_conv(x, taps, channels, [&](auto t, auto k, auto v) {
        if (p.mask)
            hipLaunchKernelGGL((conv_fwd_kernel<decltype(t), decltype(k)::value,
                                decltype(v)::value, true>), dim3(n), dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL((conv_fwd_kernel<decltype(t), decltype(k)::value,
                                decltype(v)::value, false>), dim3(n), dim3(256), 0, stream, p);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return {y, last};
}

class CausalConv : public torch::autograd::Function<CausalConv> {
public:
    static torch::autograd::variable_list forward(
        torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w,
        const OptTensor& bias_in, const OptTensor& state_in, const OptTensor& mask_in, bool silu)
    {
        const auto bias = bias_in.value_or(Tensor()), state = state_in.value_or(Tensor()),
                   mask = mask_in.value_or(Tensor());
        ctx->save_for_backward({x, w, bias, state, mask});
        const c10::DeviceGuard guard(x.device());
        ctx->saved_data["silu"] = silu;
        ctx->saved_data["capture"] = capture_now();
        ctx->set_materialize_grads(false);
        return conv_forward(x, w, bias, state, mask, silu);
    }

    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        TORCH_CHECK(!at::GradMode::is_enabled(),
                    "causal_conv: its gradients are not differentiable again");
        auto saved = ctx->get_saved_variables();
        const auto &x = saved[0], &w = saved[1], &bias = saved[2], &state = saved[3];
        const c10::DeviceGuard guard(x.device());
        check_capture("causal_conv", ctx->saved_data["capture"].toInt());
        auto stream = at::cuda::getCurrentCUDAStream();
        const int64_t taps = w.size(1);
        auto dy = grads[0].defined() ? grads[0].contiguous()
                                     : torch::zeros(x.sizes(), x.options());
        auto dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
        auto dx = torch::empty(x.sizes(), x.options());
        auto dw = torch::empty(w.sizes(), w.options());
        auto db = bias.defined() ? torch::empty({x.size(2)}, w.options()) : Tensor();
        auto dstate = state.defined() ? torch::empty(state.sizes(), x.options()) : Tensor();
        ConvArgs p = conv_args(x, w, bias, state, saved[4], ctx->saved_data["silu"].toBool());
        p.dy = ptr(dy); p.dlast = ptr(dlast); p.y = dx.data_ptr();
        p.last = dstate.defined() ? dstate.data_ptr() : nullptr;
        if (p.batch == 0 || p.steps == 0) {
            dw.zero_();
            if (db.defined()) db.zero_();
            if (dstate.defined()) {
                if (dlast.defined()) dstate.copy_(dlast); else dstate.zero_();
            }
            return {dx, dw, db, dstate, Tensor(), Tensor()};
        }
        const int channels = conv_channels(x, {state, dy, dlast});
        cut_conv(p, channels);
        // 2^17 lanes where the tiles give them, in 256 to 1024 parts (on the GPU fp32
        // 33x774x228 133 us with 2^15 lanes, 91 with 2^16, 86 with 2^17 or 2^18).
        const int64_t want = (1 << 17) / (p.width / channels);
        p.nparts = (int)std::min<int64_t>(p.batch * p.tiles,
                                          std::clamp<int64_t>(want, 256, 1024));
        auto parts = torch::empty({p.nparts, taps + 1, x.size(2)}, w.options());
        p.parts = parts.data_ptr<float>();
        by_conv(x, taps, channels, [&](auto t, auto k, auto v) {
            const int64_t n = blocks_for((int64_t)p.nparts * (p.width / v.value), "causal_conv");
            if (p.mask)
                hipLaunchKernelGGL((conv_bwd_kernel<decltype(t), decltype(k)::value,
                                    decltype(v)::value, true>), dim3(n), dim3(256), 0, stream, p);
            else
                hipLaunchKernelGGL((conv_bwd_kernel<decltype(t), decltype(k)::value,
                                    decltype(v)::value, false>), dim3(n), dim3(256), 0, stream, p);
        });
        auto rest = db.defined() ? db : torch::empty({x.size(2)}, w.options());
        const int64_t cols = (taps + 1) * x.size(2);
        hipLaunchKernelGGL(column_sum_kernel, dim3((cols + 15) / 16), dim3(256), 0, stream,
                           p.parts, (long)p.nparts, (long)p.width, (int)taps,
                           dw.data_ptr<float>(), rest.data_ptr<float>());
        C10_HIP_KERNEL_LAUNCH_CHECK();
        return {dx, dw, db, dstate, Tensor(), Tensor()};
    }
};

void check_conv(const char* op, const Tensor& x, const Tensor& w, const OptTensor& bias)
{
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) >= 2 && w.size(1) <= 4, op,
                      ": weight must be (channels, taps) with 2 to 4 taps, got ", w.sizes());
    check_like(op, "weight", w, x, torch::kFloat32, {x.size(-1), w.size(1)});
    if (bias) check_like(op, "bias", *bias, x, torch::kFloat32, {x.size(-1)});
}

bool wants_grad(std::initializer_list<OptTensor> all)
{
    if (!at::GradMode::is_enabled()) return false;
    for (auto& t : all)
        if (t && t->requires_grad()) return true;
    return false;
}

// Parameters are read as they lie, dense and on 16 byte borders.
Tensor dense(const Tensor& t)
{
    auto d = t.contiguous();
    return (uintptr_t)d.data_ptr() % 16 ? d.clone() : d;
}
OptTensor dense(const OptTensor& t) { return t ? c10::make_optional(dense(*t)) : t; }

std::vector<Tensor> causal_conv(const Tensor& x_in, const Tensor& w, const OptTensor& bias,
                                const OptTensor& state, const OptTensor& mask, bool silu)
{
    const char* op = "causal_conv";
    check_forward_mode(op, {x_in, w, bias, state});
    check_x(op, x_in, 3);
    check_conv(op, x_in, w, bias);
    if (state)
        check_like(op, "state", *state, x_in, x_in.scalar_type(),
                   {x_in.size(0), w.size(1) - 1, x_in.size(2)});
    const auto x = dense_last(x_in);
    const auto m = as_mask(op, mask, x);
    if (wants_grad({x, w, bias, state}))
        return CausalConv::apply(x, dense(w), dense(bias), dense(state),
                                 m.defined() ? OptTensor(m) : OptTensor(), silu);
    return conv_forward(x, dense(w), dense(bias).value_or(Tensor()),
                        dense(state).value_or(Tensor()), m, silu);
}

Tensor causal_conv_step(Tensor state, const Tensor& x_in, const Tensor& w, const OptTensor& bias,
                        const OptTensor& mask, bool silu)
{
    const char* op = "causal_conv_step";
    check_forward_mode(op, {state, x_in, w, bias});
    check_x(op, x_in, 2);
    check_conv(op, x_in, w, bias);
    check_like(op, "state", state, x_in, x_in.scalar_type(),
               {x_in.size(0), w.size(1) - 1, x_in.size(1)});
    TORCH_CHECK_VALUE(state.is_contiguous(), op, ": state must be contiguous");
    TORCH_CHECK_VALUE(!wants_grad({x_in, w, bias, state}), op,
                      ": has no gradient; use causal_conv over one step");
    const auto x = dense_last(x_in);
    const auto m = as_mask(op, mask, x);
    const c10::DeviceGuard guard(x.device());
    auto y = torch::empty(x.sizes(), x.options());
    if (x.size(0) == 0) return y;
    const auto wc = dense(w), bc = dense(bias).value_or(Tensor());
    ConvArgs p = conv_args(x, wc, bc, Tensor(), m, silu);
    p.y = y.data_ptr(); p.last = state.data_ptr();
    p.tile = p.batch * p.width < 1 << 20 ? 1 : CU;
    by_conv(x, w.size(1), conv_channels(x, {state}), [&](auto t, auto k, auto v) {
        const int64_t n = blocks_for((p.batch + p.tile - 1) / p.tile * (p.width / v.value), op);
        hipLaunchKernelGGL((conv_step_kernel<decltype(t), decltype(k)::value,
                            decltype(v)::value>), dim3(n), dim3(256), 0,
                           at::cuda::getCurrentCUDAStream(), p);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    moved_on(state);
    return y;
}

// ---- scan

int lanes_for(int64_t states)
{
    int l = 1;
    while (4 * l < states) l *= 2;
    return l;
}
template <typename F> void by_lanes(int l, F f)
{
    if (l == 1) f(Const<1>());
    else if (l == 2) f(Const<2>());
    else if (l == 4) f(Const<4>());
    else if (l == 8) f(Const<8>());
    else f(Const<16>());
}
template <typename F> void by_scan(const Tensor& x, int l, F f)
{
    by_type(x, [&](auto t) { by_lanes(l, [&](auto n) { f(t, n); }); });
}

struct ScanIn {
    Tensor x, dt, A, B, C, D, z, bias, state, mask;
    bool softplus;
};

// Cuts the steps into segments that run side by side where rows and channels
// alone leave the card idle; their states are joined by one more pass.
void cut_steps(ScanArgs& p)
{
    // 1024 blocks are four waves a SIMD.  1x8192x1024 forward: 370 us with 128
    // blocks, 194 with 256, 119 with 512, 97 with 1024, 96 with 2048;
    // 4x2048x2048 training: 1624, 1180, 695, 593 and 589 us.
    const int64_t target = 1024;
    const int64_t blocks = std::max<int64_t>(1, p.batch * p.groups * p.tiles);
    int64_t segs = std::max<int64_t>(1, std::min({target / blocks, p.chunks, (int64_t)64}));
    p.seg_chunks = (int)std::max<int64_t>(1, (p.chunks + segs - 1) / segs);
    // Segments are walked twice, so they have to be shorter than half of the steps.
    // On the GPU, training with and without: 100x80x256 111 and 76 us (two
    // segments of 3 of 5 chunks), 37x67x200 82 and 76 (of 2 of 5), 4x64x200 34
    // and 48 (of 1 of 4), 32x80x256 56 and 58 (of 1 of 5).
    if (2 * p.seg_chunks + 1 >= p.chunks) p.seg_chunks = (int)std::max<int64_t>(1, p.chunks);
    p.segs = (unsigned)std::max<int64_t>(1, (p.chunks + p.seg_chunks - 1) / p.seg_chunks);
}

ScanArgs scan_args(const ScanIn& s)
{
    ScanArgs p{};
    p.x = ptr(s.x); p.dt = ptr(s.dt); p.z = ptr(s.z); p.B = ptr(s.B); p.C = ptr(s.C);
    p.A = fptr(s.A); p.D = fptr(s.D); p.bias = fptr(s.bias); p.state = fptr(s.state);
    p.mask = mptr(s.mask);
    p.batch = s.x.size(0); p.steps = s.x.size(1); p.chunks = (p.steps + TC - 1) / TC;
    p.xb = s.x.stride(0); p.xt = s.x.stride(1);
    p.db = s.dt.stride(0); p.dt_ = s.dt.stride(1);
    if (s.z.defined()) { p.zb = s.z.stride(0); p.zt = s.z.stride(1); }
    p.Bb = s.B.stride(0); p.Bt = s.B.stride(1); p.Bg = s.B.stride(2);
    p.Cb = s.C.stride(0); p.Ct = s.C.stride(1); p.Cg = s.C.stride(2);
    p.width = (int)s.x.size(2); p.states = (int)s.A.size(1); p.groups = (unsigned)s.B.size(2);
    p.per = p.width / (int)p.groups;
    const int cb = 256 / lanes_for(p.states);
    p.tiles = (p.per + cb - 1) / cb;
    cut_steps(p);
    p.softplus = s.softplus;
    p.vec_d = p.per % 4 == 0 && aligned(s.x, 4) && aligned(s.dt, 4) &&
              (!s.z.defined() || aligned(s.z, 4));
    p.vec_n = p.states % 4 == 0 && aligned(s.A, 4) && (!s.state.defined() || aligned(s.state, 4));
    p.vec_b = p.states % 4 == 0 && aligned(s.B, 4) && aligned(s.C, 4);
    return p;
}

int64_t scan_blocks(const ScanArgs& p)
{
    return blocks_for(p.batch * p.segs * p.groups * p.tiles * 256, "selective_scan");
}

// What the segments hand on: a state and the sum of their steps.
Tensor segment_buffers(ScanArgs& p, const torch::TensorOptions& fp32)
{
    if (p.segs == 1) return Tensor();
    const int64_t rows = p.batch * p.segs * p.width;
    auto t = torch::empty({rows * (p.states + 1)}, fp32);
    p.seg_h = t.data_ptr<float>();
    p.seg_d = p.seg_h + rows * p.states;
    return t;
}

// y, last state and, to train, the state before each chunk
std::vector<Tensor> scan_forward(const ScanIn& s, bool train)
{
    const c10::DeviceGuard guard(s.x.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    ScanArgs p = scan_args(s);
    const int64_t blocks = scan_blocks(p);
    auto fp32 = s.A.options();
    auto y = torch::empty(s.x.sizes(), s.x.options());
    auto last = torch::empty({p.batch, p.width, p.states}, fp32);
    auto ckpt = train ? torch::empty({p.batch, p.chunks * (TC / TH), p.width, p.states}, fp32) : Tensor();
    if (p.batch == 0 || p.steps == 0) {
        if (s.state.defined()) last.copy_(s.state); else last.zero_();
        return {y, last, ckpt};
    }
    p.y = y.data_ptr(); p.last = last.data_ptr<float>();
    p.ckpt = train ? ckpt.data_ptr<float>() : nullptr;
    const auto seg = segment_buffers(p, fp32);
    by_scan(s.x, lanes_for(p.states), [&](auto t, auto n) {
        if (p.segs > 1)
            hipLaunchKernelGGL((scan_fwd_kernel<decltype(t), decltype(n)::value, true>),
                               dim3(blocks), dim3(256), 0, stream, p);
        hipLaunchKernelGGL((scan_fwd_kernel<decltype(t), decltype(n)::value, false>),
                           dim3(blocks), dim3(256), 0, stream, p);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return {y, last, ckpt};
}

class SelectiveScan : public torch::autograd::Function<SelectiveScan> {
public:
    static torch::autograd::variable_list forward(
        torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A,
        const Tensor& B, const Tensor& C, const OptTensor& D, const OptTensor& z,
        const OptTensor& bias, const OptTensor& state, const OptTensor& mask, bool softplus)
    {
        const Tensor none;
        ScanIn s{x, dt, A, B, C, D.value_or(none), z.value_or(none), bias.value_or(none),
                 state.value_or(none), mask.value_or(none), softplus};
        auto out = scan_forward(s, true);
        ctx->save_for_backward({s.x, s.dt, s.A, s.B, s.C, s.D, s.z, s.bias, s.state, s.mask,
                                out[2]});
        const c10::DeviceGuard guard(x.device());
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["capture"] = capture_now();
        ctx->set_materialize_grads(false);
        return {out[0], out[1]};
    }

    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        TORCH_CHECK(!at::GradMode::is_enabled(),
                    "selective_scan: its gradients are not differentiable again");
        auto v = ctx->get_saved_variables();
        ScanIn s{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9],
                 ctx->saved_data["softplus"].toBool()};
        const auto& ckpt = v[10];
        const c10::DeviceGuard guard(s.x.device());
        check_capture("selective_scan", ctx->saved_data["capture"].toInt());
        auto stream = at::cuda::getCurrentCUDAStream();
        ScanArgs p = scan_args(s);
        auto fp32 = s.A.options();
        auto like = [](const Tensor& t) { return torch::empty(t.sizes(), t.options()); };
        auto dy = grads[0].defined() ? grads[0].contiguous()
                                     : torch::zeros(s.x.sizes(), s.x.options());
        auto dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
        auto dx = like(s.x), ddt = like(s.dt), dA = like(s.A), dB = like(s.B), dC = like(s.C);
        auto dD = torch::empty({2, p.width}, fp32);
        auto dz = s.z.defined() ? like(s.z) : Tensor();
        auto dstate = s.state.defined() ? like(s.state) : Tensor();
        torch::autograd::variable_list out(11);
        out[0] = dx; out[1] = ddt; out[2] = dA; out[3] = dB; out[4] = dC;
        if (s.D.defined()) out[5] = dD[0];
        out[6] = dz;
        if (s.bias.defined()) out[7] = dD[1];
        out[8] = dstate;
        if (p.batch == 0 || p.steps == 0) {
            dA.zero_(); dD.zero_();
            if (dstate.defined()) {
                if (dlast.defined()) dstate.copy_(dlast); else dstate.zero_();
            }
            return out;
        }
        const int64_t rows = p.batch * p.segs, nb = dB.numel();
        // sums over tiles, rows and segments to come, in one piece
        const int64_t nA = dA.numel(), nD = dD.numel();
        auto parts = torch::empty({2 * (int64_t)p.tiles * nb + rows * (nA + nD)}, fp32);
        p.dy = ptr(dy); p.dlast = fptr(dlast);
        p.vec_d = p.vec_d && aligned(dy, 4);
        p.vec_n = p.vec_n && (!dlast.defined() || aligned(dlast, 4));
        p.ckpt = ckpt.data_ptr<float>();
        p.dx = dx.data_ptr(); p.ddt = ddt.data_ptr(); p.dz = dz.defined() ? dz.data_ptr() : nullptr;
        p.dAp = parts.data_ptr<float>(); p.dDp = p.dAp + rows * nA;
        p.dBp = p.dDp + rows * nD; p.dCp = p.dBp + p.tiles * nb;
        p.dstate = dstate.defined() ? dstate.data_ptr<float>() : nullptr;
        const auto seg = segment_buffers(p, fp32);
        by_scan(s.x, lanes_for(p.states), [&](auto t, auto n) {
            using T = decltype(t);
            if (p.segs > 1)
                hipLaunchKernelGGL((scan_bwd_kernel<T, decltype(n)::value, true>),
                                   dim3(scan_blocks(p)), dim3(256), 0, stream, p);
            hipLaunchKernelGGL((scan_bwd_kernel<T, decltype(n)::value, false>),
                               dim3(scan_blocks(p)), dim3(256), 0, stream, p);
            const int64_t blocks = 2 * ((nb + 255) / 256) + (nA + 15) / 16 + (nD + 15) / 16;
            for (int64_t first = 0; first < blocks; first += kMostBlocks)
                hipLaunchKernelGGL(scan_finish_kernel<T>,
                                   dim3(std::min(kMostBlocks, blocks - first)), dim3(256), 0,
                                   stream, p.dBp, (int)p.tiles, (long)nb, (T*)dB.data_ptr(),
                                   (T*)dC.data_ptr(), p.dAp, p.dDp, (long)rows, (long)nA,
                                   (long)nD, dA.data_ptr<float>(), dD.data_ptr<float>(),
                                   (long)first);
        });
        C10_HIP_KERNEL_LAUNCH_CHECK();
        return out;
    }
};

void check_scan(const char* op, const Tensor& x, const Tensor& dt, const Tensor& A,
                const Tensor& B, const Tensor& C, const OptTensor& D, const OptTensor& z,
                const OptTensor& bias)
{
    const auto type = x.scalar_type();
    check_like(op, "dt", dt, x, type, x.sizes());
    TORCH_CHECK_VALUE(A.dim() == 2 && A.size(1) >= 1 && A.size(1) <= 64, op,
                      ": A must be (channels, states) with 1 to 64 states, got ", A.sizes());
    check_like(op, "A", A, x, torch::kFloat32, {x.size(-1), A.size(1)});
    auto shape = x.sizes().slice(0, x.dim() - 1).vec();
    TORCH_CHECK_VALUE(B.dim() == x.dim() + 1 && B.size(-2) >= 1 &&
                      x.size(-1) % B.size(-2) == 0, op,
                      ": B must be (..., groups, states) with groups that divide the channels, got ",
                      B.sizes());
    shape.push_back(B.size(-2));
    shape.push_back(A.size(1));
    check_like(op, "B", B, x, type, shape);
    check_like(op, "C", C, x, type, shape);
    if (D) check_like(op, "D", *D, x, torch::kFloat32, {x.size(-1)});
    if (z) check_like(op, "z", *z, x, type, x.sizes());
    if (bias) check_like(op, "dt_bias", *bias, x, torch::kFloat32, {x.size(-1)});
}

std::vector<Tensor> selective_scan(
    const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
    const OptTensor& D, const OptTensor& z, const OptTensor& bias, bool softplus,
    const OptTensor& state, const OptTensor& mask)
{
    const char* op = "selective_scan";
    check_forward_mode(op, {x, dt, A, B, C, D, z, bias, state});
    check_x(op, x, 3);
    check_scan(op, x, dt, A, B, C, D, z, bias);
    if (state)
        check_like(op, "state", *state, x, torch::kFloat32, {x.size(0), x.size(2), A.size(1)});
    const auto m = as_mask(op, mask, x);
    const Tensor none;
    const auto zd = z ? OptTensor(dense_last(*z)) : z;
    ScanIn s{dense_last(x), dense_last(dt), dense(A), dense_last(B), dense_last(C),
             dense(D).value_or(none), zd.value_or(none), dense(bias).value_or(none),
             dense(state).value_or(none), m, softplus};
    if (wants_grad({x, dt, A, B, C, D, z, bias, state}))
        return SelectiveScan::apply(s.x, s.dt, s.A, s.B, s.C, dense(D), zd, dense(bias),
                                    dense(state), m.defined() ? OptTensor(m) : OptTensor(),
                                    softplus);
    auto out = scan_forward(s, false);
    return {out[0], out[1]};
}

Tensor selective_step(Tensor state, const Tensor& x_in, const Tensor& dt_in, const Tensor& A_in,
                      const Tensor& B_in, const Tensor& C_in, const OptTensor& D_in,
                      const OptTensor& z_in, const OptTensor& bias_in, bool softplus,
                      const OptTensor& mask)
{
    const char* op = "selective_step";
    check_forward_mode(op, {state, x_in, dt_in, A_in, B_in, C_in, D_in, z_in, bias_in});
    check_x(op, x_in, 2);
    check_scan(op, x_in, dt_in, A_in, B_in, C_in, D_in, z_in, bias_in);
    check_like(op, "state", state, x_in, torch::kFloat32,
               {x_in.size(0), x_in.size(1), A_in.size(1)});
    TORCH_CHECK_VALUE(state.is_contiguous(), op, ": state must be contiguous");
    TORCH_CHECK_VALUE(!wants_grad({x_in, dt_in, A_in, B_in, C_in, D_in, z_in, bias_in, state}),
                      op, ": has no gradient; use selective_scan over one step");
    const auto m = as_mask(op, mask, x_in);
    const c10::DeviceGuard guard(x_in.device());
    auto y = torch::empty(x_in.sizes(), x_in.options());
    if (x_in.size(0) == 0) return y;
    const Tensor none;
    const auto x = dense_last(x_in), dt = dense_last(dt_in), A = dense(A_in),
               B = dense_last(B_in), C = dense_last(C_in), D = dense(D_in).value_or(none),
               z = z_in ? dense_last(*z_in) : none, bias = dense(bias_in).value_or(none);
    StepArgs p{};
    p.x = ptr(x); p.dt = ptr(dt); p.z = ptr(z); p.B = ptr(B); p.C = ptr(C);
    p.A = fptr(A); p.D = fptr(D); p.bias = fptr(bias); p.mask = mptr(m);
    p.state = state.data_ptr<float>(); p.y = y.data_ptr();
    p.batch = x.size(0); p.xb = x.stride(0); p.db = dt.stride(0);
    p.zb = z.defined() ? z.stride(0) : 0;
    p.Bb = B.stride(0); p.Bg = B.stride(1); p.Cb = C.stride(0); p.Cg = C.stride(1);
    p.width = (int)x.size(1); p.states = (int)A.size(1); p.groups = (int)B.size(1);
    p.per = p.width / p.groups; p.softplus = softplus;
    p.vec_n = p.states % 4 == 0 && aligned(state, 4) && aligned(A, 4);
    p.vec_b = p.states % 4 == 0 && aligned(B, 4) && aligned(C, 4);
    const int l = lanes_for(p.states);
    p.rows = p.batch * p.width * l < 1 << 20 ? 1 : SR;
    const int64_t n = blocks_for((p.batch + p.rows - 1) / p.rows * p.width * l, op);
    by_scan(x, l, [&](auto t, auto k) {
        hipLaunchKernelGGL((scan_step_kernel<decltype(t), decltype(k)::value>), dim3(n),
                           dim3(256), 0, at::cuda::getCurrentCUDAStream(), p);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    moved_on(state);
    return y;
}

}  // namespace

void bind_selective(pybind11::module& m)
{
    m.def("causal_conv", &causal_conv, "short causal convolution over a window (y, last state)");
    m.def("causal_conv_step", &causal_conv_step, "one step of it, the state in place");
    m.def("selective_scan", &selective_scan, "selective state space scan (y, last state)");
    m.def("selective_step", &selective_step, "one step of it, the state in place");
}
