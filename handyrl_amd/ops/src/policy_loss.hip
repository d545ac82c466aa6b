// Clipped policy loss with a KL term and an entropy bonus over rows of
// logits, and its gradient.
//
// With lp = z[a] - lse(z), x = lp - lp_old, r = exp(x) and row weight m:
//   surrogate  s = min(r adv, clamp(r, 1 - lo, 1 + hi) adv)
//   kl         k = r - 1 - x       (estimates KL(old || new): a ~ old)
//   entropy    H = -sum_j p_j log p_j
//   loss       = sum_rows m (-s + beta k - gamma e H)
//   dloss/dz_j = c (d_ja - p_j) + w p_j (log p_j + H)
//     c = m ((s is on its flat side ? 0 : -r adv) + beta (r - 1)),
//     w = m gamma e
// Rows of weight 0 are not read: they give nothing to the sums and a zero
// gradient, whatever their logits hold.

#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <hip/hip_runtime.h>
#include "guards.h"

namespace {

constexpr int kStats = 6;       // -m s, m k, m H, m e H, clipped rows, m
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e4f;   // behind it e^x is 0; keeps 0 * inf out of sums

struct LossArgs {
    const void* logits;         // (R, A), rows `stride` apart
    const long* action;
    const float* old_lp;
    const float* adv;
    const float* mask;          // null: all ones
    const float* escale;        // null: all ones
    void* grad;                 // (R, A) dense, or null
    double* partial;            // (blocks, kStats), or null: backward
    const float* upstream;      // null: 1
    int skip_one;               // the gradient stands there already if upstream is 1
    long rows, stride;
    int width;
    float lo, hi, beta, gamma;
};

using bf16 = __hip_bfloat16;
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16(v); }

// Reductions over G neighbouring lanes; every lane gets the result.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
        0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
struct Sum { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
template <int G, typename F> __device__ __forceinline__ float over_lanes(float v, F f) {
    if (G > 1) v = f(v, dpp<0xB1>(v));          // quad lanes 1 0 3 2
    if (G > 2) v = f(v, dpp<0x4E>(v));          // quad lanes 2 3 0 1
    if (G > 4) v = f(v, dpp<0x141>(v));         // the half row backwards
    if (G > 8) v = f(v, dpp<0x140>(v));         // the row backwards
    if (G > 16) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const unsigned x = r[0], y = r[1];
        v = f(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
    }
    if (G > 32) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const unsigned x = r[0], y = r[1];
        v = f(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
    }
    return v;
}

// e^x with the rounding of x log2(e) made good, and e^x - 1 - x, by its series
// where that subtraction would cancel (the term left out is below 2^-24 of it).
__device__ __forceinline__ float exp_of(float x) {
    const float t = x * kLog2e;
    const float rest = fmaf(x, kLog2e, -t) + x * 1.925963033500e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fabsf(x) < 80.f ? fmaf(e, rest * 0.69314718f, e) : e;
}
__device__ __forceinline__ float exp_rest(float x, float exp_x) {
    float s = 1.f / 3628800.f;
    s = fmaf(s, x, 1.f / 362880.f);
    s = fmaf(s, x, 1.f / 40320.f);
    s = fmaf(s, x, 1.f / 5040.f);
    s = fmaf(s, x, 1.f / 720.f);
    s = fmaf(s, x, 1.f / 120.f);
    s = fmaf(s, x, 1.f / 24.f);
    s = fmaf(s, x, 1.f / 6.f);
    s = fmaf(s, x, 0.5f) * x * x;
    return fabsf(x) < 1.f ? s : exp_x - 1.f - x;
}

// What a row's gradient needs: dz_j = e (slope max(x, kFar) + level) and `pull`
// more for the taken action, with x = z_j - top, e = e^x.
struct Row {
    float top, slope, level, pull;
    float surrogate, kl, entropy, clipped;
};

// From S0 = sum e and S1 = sum e x.
__device__ __forceinline__ Row row_terms(const LossArgs& p, float m, float escale, float old_lp,
                                         float adv, float top, float s0, float s1,
                                         float z_a) {
    Row r;
    const float log_sum = __builtin_amdgcn_logf(s0) * 0.69314718056f;
    const float inv = __builtin_amdgcn_rcpf(s0);
    const float x = (z_a - top) - log_sum - old_lp;
    const float ratio = exp_of(x);
    const float bound = fminf(fmaxf(ratio, 1.f - p.lo), 1.f + p.hi);
    const bool flat = (adv > 0.f && ratio > 1.f + p.hi) ||
                      (adv < 0.f && ratio < 1.f - p.lo);
    r.top = top;
    r.entropy = log_sum - s1 * inv;
    r.surrogate = flat ? bound * adv : ratio * adv;
    r.kl = exp_rest(x, ratio);
    r.clipped = flat ? 1.f : 0.f;
    r.pull = m * ((flat ? 0.f : -ratio * adv) +
                  (p.beta != 0.f ? p.beta * (ratio - 1.f) : 0.f));      // not 0 * inf
    // with p_j = e / S0 and log p_j = x - log S0:
    //   -pull p_j + w p_j (log p_j + H) = e / S0 (w x + w (H - log S0) - pull)
    const float w = m * p.gamma * escale;
    r.slope = w * inv;
    r.level = (w * (r.entropy - log_sum) - r.pull) * inv;
    return r;
}

__device__ __forceinline__ float row_grad(const Row& r, float z) {
    const float x = z - r.top;
    return __builtin_amdgcn_exp2f(x * kLog2e) * fmaf(r.slope, fmaxf(x, kFar), r.level);
}

struct RowIn {
    float m, escale, old_lp, adv;
    int a;                              // -1: not an action
    __device__ __forceinline__ RowIn(const LossArgs& p, long i) {
        m = p.mask ? p.mask[i] : 1.f;
        escale = p.escale ? p.escale[i] : 1.f;
        old_lp = p.old_lp[i];
        adv = p.adv[i];
        const long at = p.action[i];
        a = at >= 0 && at < p.width ? (int)at : -1;
    }
};

__device__ __forceinline__ void add_row(double* sum, const Row& r, const RowIn& in) {
    const double m = in.m;
    sum[0] -= m * r.surrogate;
    sum[1] += m * r.kl;
    sum[2] += m * r.entropy;
    sum[3] += m * in.escale * r.entropy;
    sum[4] += r.clipped;
    sum[5] += m;
}

// Rows of up to 64 E values: G lanes a row, the row in registers, E a lane.
// 16384x214 fp32: 12 us with the gradient (28 MB; launch and latency are 3 of
// them), 13 + 13 with a kernel each way that reads the row three times.
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void policy_rows_kernel(LossArgs p)
{
    const float up = p.upstream ? p.upstream[0] : 1.f;
    if (p.skip_one && up == 1.f) return;
    constexpr int per = 256 / G;
    const int sub = threadIdx.x % G;
    double sum[kStats] = {};
    // all lanes walk alike, since the reductions need whole waves
    for (long i0 = (long)blockIdx.x * per; i0 < p.rows; i0 += (long)gridDim.x * per) {
        const long i = i0 + threadIdx.x / G;
        const bool there = i < p.rows;
        const RowIn in(p, there ? i : p.rows - 1);
        const bool on = there && in.m != 0.f;
        const T* row = (const T*)p.logits + (there ? i : 0) * p.stride;
        float z[E], top = -INFINITY, z_a = NAN;
        if (on && in.a >= 0) z_a = to_float(row[in.a]);
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int j = sub + k * G;
            z[k] = on && j < p.width ? to_float(row[j]) : -INFINITY;
            top = fmaxf(top, z[k]);
        }
        top = over_lanes<G>(top, Max());
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const float x = z[k] - top, e = __builtin_amdgcn_exp2f(x * kLog2e);
            // behind the row's end z is -inf, and e 0 (but not beside a top of -inf)
            s0 += sub + k * G < p.width ? e : 0.f;
            s1 += sub + k * G < p.width ? e * fmaxf(x, kFar) : 0.f;
        }
        s0 = over_lanes<G>(s0, Sum());
        s1 = over_lanes<G>(s1, Sum());
        const Row r = row_terms(p, in.m, in.escale, in.old_lp, in.adv, top, s0, s1, z_a);
        if (p.grad && there) {
            T* out = (T*)p.grad + i * p.width;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const int j = sub + k * G;
                float d = row_grad(r, z[k]);
                if (j == in.a) d += r.pull;
                if (j < p.width) out[j] = from_float<T>(on ? up * d : 0.f);
            }
        }
        if (on && sub == 0) add_row(sum, r, in);
    }
    if (!p.partial) return;
    __shared__ double fold[per][kStats];
    if (sub == 0)
        for (int k = 0; k < kStats; ++k) fold[threadIdx.x / G][k] = sum[k];
    __syncthreads();
    if (threadIdx.x < kStats) {
        double s = 0;
        for (int i = 0; i < per; ++i) s += fold[i][threadIdx.x];
        p.partial[(long)blockIdx.x * kStats + threadIdx.x] = s;
    }
}

// Reductions over a block of NT threads; `fold` holds a value a wave.
template <int NT, typename F>
__device__ __forceinline__ float over_block(float v, F f, float* fold) {
    v = over_lanes<64>(v, f);
    if ((threadIdx.x & 63) == 0) fold[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = fold[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) r = f(r, fold[i]);
    return r;
}

// 16 bytes of values, held as the four words that they are.
template <typename T> struct Vec {
    static constexpr int n = 16 / sizeof(T);
    typedef unsigned __attribute__((ext_vector_type(4))) words;
    words w;
    __device__ __forceinline__ float get(int q) const {
        if (sizeof(T) == 4) return __builtin_bit_cast(float, (unsigned)w[q]);
        const unsigned u = w[q / 2];
        return __builtin_bit_cast(float, q % 2 ? u & 0xffff0000u : u << 16);
    }
    __device__ __forceinline__ static Vec of(const float* d) {
        Vec r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (sizeof(T) == 4) {
                r.w[i] = __builtin_bit_cast(unsigned, d[i]);
            } else {
                const unsigned short lo = __builtin_bit_cast(unsigned short, from_float<bf16>(d[2 * i]));
                const unsigned short hi = __builtin_bit_cast(unsigned short, from_float<bf16>(d[2 * i + 1]));
                r.w[i] = lo | (unsigned)hi << 16;
            }
        }
        return r;
    }
    // Keeps the compiler from holding the values as floats from one use to the
    // next, which takes twice the registers.
    __device__ __forceinline__ void stay_packed() { asm volatile("" : "+v"(w)); }
};

// Wide rows, a block a row.  What lies between the row's 16 byte borders is
// taken 16 bytes a lane at a time: CH such pieces a lane stay in registers, so
// that the row is read once; CH = 0 walks rows of any width and reads them
// again.  The few values before the first border and behind the last are one
// more value each for the first lanes.  Memory bounds it: 4096x32003 bf16 takes
// 123 us with the gradient, 4.3 TB/s where a copy reaches 5.1 (1036 us in two
// kernels that read the row seven times).
template <typename T, int NT, int CH>
__global__ __launch_bounds__(NT, 1024 / NT) void policy_wide_kernel(LossArgs p)
{
    const float up = p.upstream ? p.upstream[0] : 1.f;
    if (p.skip_one && up == 1.f) return;
    constexpr int V = Vec<T>::n;
    __shared__ float fold[3][NT / 64];
    __shared__ double sum[kStats];      // the first lane's
    const int tid = threadIdx.x;
    if (tid == 0)
        for (int k = 0; k < kStats; ++k) sum[k] = 0;
    for (long i = blockIdx.x; i < p.rows; i += gridDim.x) {
        const RowIn in(p, i);
        const T* row = (const T*)p.logits + i * p.stride;
        T* out = p.grad ? (T*)p.grad + i * p.width : nullptr;
        const int head = min(p.width, (int)((V - (uintptr_t)row / sizeof(T) % V) % V));
        const int pieces = (p.width - head) / V, tail = head + pieces * V;
        const int edge = tid < head ? tid : tid >= V && tid - V < p.width - tail ? tail + tid - V : -1;
        const auto* body = (const typename Vec<T>::words*)(row + head);
        T* to = out + head;
        const bool even = ((uintptr_t)row - (uintptr_t)out) % 16 == 0;
        auto store = [&](int c, const float* d) {
            if (even) {
                *(typename Vec<T>::words*)(to + c * V) = Vec<T>::of(d).w;
            } else {
#pragma unroll
                for (int q = 0; q < V; ++q) to[c * V + q] = from_float<T>(d[q]);
            }
        };
        if (in.m == 0.f) {              // not read at all
            const float none[V] = {};
            if (out) {
                for (int c = tid; c < pieces; c += NT) store(c, none);
                if (edge >= 0) out[edge] = from_float<T>(0.f);
            }
            continue;
        }
        const float z_a = in.a >= 0 ? to_float(row[in.a]) : NAN;
        Vec<T> keep[CH > 0 ? CH : 1];
        const float z_edge = edge >= 0 ? to_float(row[edge]) : -INFINITY;
        float top = z_edge, s0 = 0.f, s1 = 0.f;
        if (CH > 0) {
#pragma unroll
            for (int k = 0; k < CH; ++k)
                if (tid + k * NT < pieces) keep[k].w = body[tid + k * NT];
        }
        // the lane's pieces, one after the other
        auto each = [&](auto f) {
            if (CH > 0) {
#pragma unroll
                for (int k = 0; k < CH; ++k)
                    if (tid + k * NT < pieces) {
                        keep[k].stay_packed();
                        f(keep[k], tid + k * NT);
                    }
            } else {
                for (int c = tid; c < pieces; c += NT) f(Vec<T>{body[c]}, c);
            }
        };
        each([&](const Vec<T>& w, int) {
#pragma unroll
            for (int q = 0; q < V; ++q) top = fmaxf(top, w.get(q));
        });
        top = over_block<NT>(top, Max(), fold[0]);
        auto add = [&](float z) {
            const float x = z - top, e = __builtin_amdgcn_exp2f(x * kLog2e);
            s0 += e;
            s1 = fmaf(e, fmaxf(x, kFar), s1);
        };
        if (edge >= 0) add(z_edge);
        each([&](const Vec<T>& w, int) {
#pragma unroll
            for (int q = 0; q < V; ++q) add(w.get(q));
        });
        s0 = over_block<NT>(s0, Sum(), fold[1]);
        s1 = over_block<NT>(s1, Sum(), fold[2]);
        const Row r = row_terms(p, in.m, in.escale, in.old_lp, in.adv, top, s0, s1, z_a);
        if (out) {
            each([&](const Vec<T>& w, int c) {
                float d[V];
#pragma unroll
                for (int q = 0; q < V; ++q) d[q] = row_grad(r, w.get(q));
                const int q_a = in.a - head - c * V;
                if (q_a >= 0 && q_a < V)
#pragma unroll
                    for (int q = 0; q < V; ++q)
                        if (q == q_a) d[q] += r.pull;
#pragma unroll
                for (int q = 0; q < V; ++q) d[q] *= up;
                store(c, d);
            });
            if (edge >= 0)
                out[edge] = from_float<T>(up * (row_grad(r, z_edge) + (edge == in.a ? r.pull : 0.f)));
        }
        if (tid == 0) add_row(sum, r, in);
        __syncthreads();                // the next row writes `fold` again
    }
    if (p.partial && tid == 0)
        for (int k = 0; k < kStats; ++k) p.partial[(long)blockIdx.x * kStats + k] = sum[k];
}

__global__ __launch_bounds__(256) void policy_loss_finish_kernel(
    const double* __restrict__ partial, int parts, float beta, float gamma,
    float* __restrict__ loss, float* __restrict__ stats)
{
    double sum[kStats] = {};
    for (int i = threadIdx.x; i < parts; i += 256)
        for (int k = 0; k < kStats; ++k) sum[k] += partial[(long)i * kStats + k];
    __shared__ double s[256][kStats];
    for (int k = 0; k < kStats; ++k) s[threadIdx.x][k] = sum[k];
    __syncthreads();
    for (int step = 128; step > 0; step >>= 1) {
        if ((int)threadIdx.x < step)
            for (int k = 0; k < kStats; ++k)
                s[threadIdx.x][k] += s[threadIdx.x + step][k];
        __syncthreads();
    }
    if (threadIdx.x < kStats) stats[threadIdx.x] = (float)s[0][threadIdx.x];
    if (threadIdx.x == 0)
        loss[0] = (float)(s[0][0] + (beta != 0.f ? (double)beta * s[0][1] : 0.) -
                          (double)gamma * s[0][3]);
}

// One value a row: `t` has the rows' shape, perhaps with a last axis of 1, or
// broadcasts to it.
torch::Tensor per_row(const torch::Tensor& t, const char* name, at::IntArrayRef rows,
                      const torch::Tensor& logits, torch::ScalarType type)
{
    TORCH_CHECK_VALUE(t.device() == logits.device(), "clipped_policy_loss: ", name,
                      " is on ", t.device(), ", logits on ", logits.device());
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && t.requires_grad()),
                      "clipped_policy_loss: ", name, " is a constant of the loss: detach it");
    TORCH_CHECK_VALUE((type == torch::kLong) == (t.scalar_type() == torch::kLong),
                      "clipped_policy_loss: ", name, " has type ", t.scalar_type());
    auto v = t;
    if (v.dim() == (int64_t)rows.size() + 1 && v.size(-1) == 1) v = v.squeeze(-1);
    if (v.sizes() != rows) {
        TORCH_CHECK_VALUE(at::is_expandable_to(v.sizes(), rows), "clipped_policy_loss: ",
                          name, " of shape ", t.sizes(), " does not fit rows of shape ", rows);
        v = v.expand(rows);
    }
    return v.to(type).contiguous();
}


LossArgs make_args(const torch::Tensor& flat, const torch::Tensor& action,
                   const torch::Tensor& old_lp, const torch::Tensor& adv,
                   const torch::Tensor& mask, const torch::Tensor& escale,
                   double lo, double hi, double beta, double gamma)
{
    LossArgs p{};
    p.logits = flat.data_ptr();
    p.action = action.data_ptr<int64_t>();
    p.old_lp = old_lp.data_ptr<float>();
    p.adv = adv.data_ptr<float>();
    p.mask = mask.defined() ? mask.data_ptr<float>() : nullptr;
    p.escale = escale.defined() ? escale.data_ptr<float>() : nullptr;
    p.rows = flat.size(0);
    p.stride = flat.stride(0);
    p.width = (int)flat.size(1);
    p.lo = (float)lo; p.hi = (float)hi; p.beta = (float)beta; p.gamma = (float)gamma;
    return p;
}

// Blocks of a launch: as many as the rows fill, each walking over several
// rows behind that, so that few partial sums are left.
int64_t blocks_of(const LossArgs& p, int64_t rows_per_block, int64_t most)
{
    return std::min((p.rows + rows_per_block - 1) / rows_per_block, most);
}

template <typename T, int G, int E> int64_t launch_rows(const LossArgs& p, hipStream_t stream,
                                                        bool count)
{
    const int64_t n = blocks_of(p, 256 / G, 1024);
    if (!count)
        hipLaunchKernelGGL((policy_rows_kernel<T, G, E>), dim3(n), dim3(256), 0, stream, p);
    return n;
}

template <typename T, int NT, int CH> int64_t launch_wide(const LossArgs& p, hipStream_t stream,
                                                          bool count)
{
    const int64_t n = blocks_of(p, 1, 2048);
    if (!count)
        hipLaunchKernelGGL((policy_wide_kernel<T, NT, CH>), dim3(n), dim3(NT), 0, stream, p);
    return n;
}

// Launches the kernel for the rows' width, or only counts its blocks.
template <typename T> int64_t launch(const LossArgs& p, hipStream_t stream, bool count)
{
    const int a = p.width;
    if (a <= 2) return launch_rows<T, 2, 1>(p, stream, count);
    if (a <= 4) return launch_rows<T, 4, 1>(p, stream, count);
    if (a <= 8) return launch_rows<T, 8, 1>(p, stream, count);
    if (a <= 16) return launch_rows<T, 16, 1>(p, stream, count);
    if (a <= 32) return launch_rows<T, 32, 1>(p, stream, count);
    if (a <= 64) return launch_rows<T, 64, 1>(p, stream, count);
    if (a <= 128) return launch_rows<T, 64, 2>(p, stream, count);
    if (a <= 256) return launch_rows<T, 64, 4>(p, stream, count);
    if (a <= 512) return launch_rows<T, 64, 8>(p, stream, count);
    if (a <= 1024) return launch_rows<T, 64, 16>(p, stream, count);
    constexpr int V = Vec<T>::n;
    const int64_t pieces = a / V;
    if (pieces <= 256 * 2) return launch_wide<T, 256, 2>(p, stream, count);
    if (pieces <= 256 * 4) return launch_wide<T, 256, 4>(p, stream, count);
    if (pieces <= 256 * 8) return launch_wide<T, 256, 8>(p, stream, count);
    if (pieces <= 512 * 8) return launch_wide<T, 512, 8>(p, stream, count);
    if (pieces <= 1024 * 8) return launch_wide<T, 1024, 8>(p, stream, count);
    return launch_wide<T, 1024, 0>(p, stream, count);
}

int64_t launch(const torch::Tensor& logits, const LossArgs& p, hipStream_t stream, bool count)
{
    if (p.rows == 0) return 0;
    const int64_t n = logits.scalar_type() == torch::kBFloat16 ? launch<bf16>(p, stream, count)
                                                                : launch<float>(p, stream, count);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return n;
}

torch::Tensor as_rows(const torch::Tensor& logits)
{
    auto flat = logits.dim() == 2 ? logits : logits.reshape({-1, logits.size(-1)});
    return flat.size(1) > 1 && flat.stride(1) != 1 ? flat.contiguous() : flat;
}

std::vector<torch::Tensor> policy_forward(
    const torch::Tensor& logits, const torch::Tensor& action, const torch::Tensor& old_lp,
    const torch::Tensor& adv, const torch::Tensor& mask, const torch::Tensor& escale,
    double lo, double hi, double beta, double gamma, bool train)
{
    const c10::DeviceGuard guard(logits.device());
    hipStream_t stream = at::cuda::getCurrentCUDAStream();
    const auto flat = as_rows(logits);
    LossArgs p = make_args(flat, action, old_lp, adv, mask, escale, lo, hi, beta, gamma);
    auto fp32 = logits.options().dtype(torch::kFloat32);
    auto loss = torch::empty({}, fp32);
    auto stats = torch::empty({kStats}, fp32);
    auto grad = train ? torch::empty(logits.sizes(), logits.options()) : torch::Tensor();
    const int64_t blocks = launch(logits, p, stream, true);
    auto partial = torch::empty({blocks, kStats}, fp32.dtype(torch::kFloat64));
    p.partial = partial.data_ptr<double>();
    p.grad = train ? grad.data_ptr() : nullptr;
    launch(logits, p, stream, false);
    hipLaunchKernelGGL(policy_loss_finish_kernel, dim3(1), dim3(256), 0, stream,
        p.partial, (int)blocks, p.beta, p.gamma, loss.data_ptr<float>(),
        stats.data_ptr<float>());
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return {loss, stats, grad};
}

// The forward pass has a row in registers when it knows what its gradient
// takes, so it writes the gradient for an upstream one of 1: the row is read
// once and written once.  The backward pass hands that out, and computes it
// anew where the upstream gradient, which only the GPU knows, is another
// number, where it has been handed out before, or where the two passes are not
// of the same captured graph and so need not run in turn.
class PolicyLoss : public torch::autograd::Function<PolicyLoss> {
public:
    static torch::autograd::variable_list forward(
        torch::autograd::AutogradContext* ctx, const torch::Tensor& logits,
        const torch::Tensor& action, const torch::Tensor& old_lp, const torch::Tensor& adv,
        const c10::optional<torch::Tensor>& mask_in,
        const c10::optional<torch::Tensor>& escale_in,
        double lo, double hi, double beta, double gamma)
    {
        const auto mask = mask_in.value_or(torch::Tensor());
        const auto escale = escale_in.value_or(torch::Tensor());
        auto out = policy_forward(logits, action, old_lp, adv, mask, escale, lo, hi, beta, gamma,
                                  true);
        ctx->save_for_backward({logits, action, old_lp, adv, mask, escale});
        ctx->saved_data["coefs"] = std::vector<double>{lo, hi, beta, gamma};
        ctx->saved_data["grad"] = out[2];
        const c10::DeviceGuard guard(logits.device());
        ctx->saved_data["capture"] = capture_now();
        ctx->mark_non_differentiable({out[1]});
        ctx->set_materialize_grads(false);
        return {out[0], out[1]};
    }

    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        TORCH_CHECK(!at::GradMode::is_enabled(),
                    "clipped_policy_loss: its gradient is not differentiable again");
        torch::autograd::variable_list out(10);
        if (!grads[0].defined()) return out;
        auto saved = ctx->get_saved_variables();
        const auto& logits = saved[0];
        const auto coefs = ctx->saved_data["coefs"].toDoubleVector();
        const c10::DeviceGuard guard(logits.device());
        hipStream_t stream = at::cuda::getCurrentCUDAStream();
        const int64_t then = ctx->saved_data["capture"].toInt();
        check_capture("clipped_policy_loss", then);
        torch::Tensor grad;
        if (!ctx->saved_data["grad"].isNone()) {
            grad = ctx->saved_data["grad"].toTensor();
            ctx->saved_data["grad"] = c10::IValue();
        }
        const bool ready = grad.defined() && then == capture_now();
        if (!ready) grad = torch::empty(logits.sizes(), logits.options());
        const auto flat = as_rows(logits);
        const auto up = grads[0].to(torch::kFloat32);
        LossArgs p = make_args(flat, saved[1], saved[2], saved[3], saved[4], saved[5],
                               coefs[0], coefs[1], coefs[2], coefs[3]);
        p.grad = grad.data_ptr();
        p.upstream = up.data_ptr<float>();
        p.skip_one = ready;
        launch(logits, p, stream, false);
        out[0] = grad;
        return out;
    }
};

std::vector<torch::Tensor> clipped_policy_loss(
    const torch::Tensor& logits, const torch::Tensor& action, const torch::Tensor& old_lp,
    const torch::Tensor& adv, const c10::optional<torch::Tensor>& mask,
    const c10::optional<torch::Tensor>& escale, double lo, double hi, double beta, double gamma)
{
    check_forward_mode("clipped_policy_loss", {logits, old_lp, adv, mask, escale});
    TORCH_CHECK_VALUE(logits.is_cuda(), "clipped_policy_loss: logits must be on the GPU");
    TORCH_CHECK_VALUE(logits.scalar_type() == torch::kFloat32 ||
                      logits.scalar_type() == torch::kBFloat16,
                      "clipped_policy_loss: logits must be float32 or bfloat16, got ",
                      logits.scalar_type());
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 &&
                      logits.size(-1) < (1L << 30),
                      "clipped_policy_loss: logits must be (..., actions), got ",
                      logits.sizes());
    auto rows = logits.sizes().slice(0, logits.dim() - 1);
    auto maybe = [&](const c10::optional<torch::Tensor>& t, const char* name) {
        return t ? c10::make_optional(per_row(*t, name, rows, logits, torch::kFloat32))
                 : c10::optional<torch::Tensor>();
    };
    const auto a = per_row(action, "actions", rows, logits, torch::kLong);
    const auto o = per_row(old_lp, "old_log_probs", rows, logits, torch::kFloat32);
    const auto d = per_row(adv, "advantages", rows, logits, torch::kFloat32);
    const auto m = maybe(mask, "mask"), e = maybe(escale, "entropy_scale");
    if (at::GradMode::is_enabled() && logits.requires_grad())
        return PolicyLoss::apply(logits, a, o, d, m, e, lo, hi, beta, gamma);
    const torch::Tensor none;
    auto out = policy_forward(logits, a, o, d, m.value_or(none), e.value_or(none), lo, hi, beta,
                              gamma, false);
    return {out[0], out[1]};
}

}  // namespace

void bind_policy_loss(pybind11::module& m)
{
    m.def("clipped_policy_loss", &clipped_policy_loss,
          "clipped policy loss with KL term and entropy bonus (loss, stats)");
}
