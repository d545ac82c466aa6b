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

namespace {

constexpr int kStats = 6;       // -m s, m k, m H, m e H, clipped rows, m

struct LossArgs {
    const void* logits;         // (R, A), rows `stride` apart
    const long* action;
    const float* old_lp;
    const float* adv;
    const float* mask;          // null: all ones
    const float* escale;        // null: all ones
    long rows, stride;
    int width;
    float lo, hi, beta, gamma;
};

__device__ __forceinline__ float load_as_float(const float* p) { return *p; }
__device__ __forceinline__ float load_as_float(const __hip_bfloat16* p) {
    return __bfloat162float(*p);
}
__device__ __forceinline__ void store_from(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_from(__hip_bfloat16* p, float v) {
    *p = __float2bfloat16(v);
}

__device__ __forceinline__ float wave_max(float v) {
    for (int s = 32; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

struct Row {
    float top, log_sum, entropy, mask, escale;
    float pull, spread;          // c and w above
    float surrogate, kl, clipped;
};

// The row's statistics from max, S0 = sum e^(z-max), S1 = sum (z-max)e^(z-max).
__device__ __forceinline__ Row row_terms(const LossArgs& p, long i, float m,
                                         float top, float s0, float s1,
                                         float z_a) {
    Row r;
    r.top = top;
    r.log_sum = logf(s0);
    r.entropy = r.log_sum - s1 / s0;
    r.mask = m;
    r.escale = p.escale ? p.escale[i] : 1.f;
    const float x = (z_a - top) - r.log_sum - p.old_lp[i];
    const float ratio = expf(x);
    const float adv = p.adv[i];
    const float bound = fminf(fmaxf(ratio, 1.f - p.lo), 1.f + p.hi);
    const bool flat = (adv > 0.f && ratio > 1.f + p.hi) ||
                      (adv < 0.f && ratio < 1.f - p.lo);
    r.surrogate = fminf(ratio * adv, bound * adv);
    if (ratio != ratio || adv != adv) r.surrogate = ratio * adv;
    r.kl = expm1f(x) - x;
    r.clipped = flat ? 1.f : 0.f;
    r.pull = m * ((flat ? 0.f : -ratio * adv) + p.beta * (ratio - 1.f));
    r.spread = m * p.gamma * r.escale;
    return r;
}

__device__ __forceinline__ float row_grad(const Row& r, float z, bool taken) {
    const float lp = (z - r.top) - r.log_sum;
    const float pj = __expf(lp);
    const float ent = pj > 0.f ? r.spread * pj * (lp + r.entropy) : 0.f;
    return r.pull * ((taken ? 1.f : 0.f) - pj) + (pj != pj ? pj : ent);
}

template <typename T>
__device__ __forceinline__ Row wave_row(const LossArgs& p, long i, float m,
                                        int lane) {
    const T* row = (const T*)p.logits + i * p.stride;
    float top = -INFINITY;
    for (int j = lane; j < p.width; j += 64)
        top = fmaxf(top, load_as_float(row + j));
    top = wave_max(top);
    float s0 = 0.f, s1 = 0.f;
    for (int j = lane; j < p.width; j += 64) {
        const float x = load_as_float(row + j) - top;
        const float e = __expf(x);
        s0 += e;
        s1 += e > 0.f ? e * x : 0.f;
    }
    s0 = wave_sum(s0);
    s1 = wave_sum(s1);
    const long a = p.action[i];
    const float z_a = a >= 0 && a < p.width ? load_as_float(row + a) : NAN;
    return row_terms(p, i, m, top, s0, s1, z_a);
}

template <typename T>
__global__ __launch_bounds__(256) void policy_loss_fwd_kernel(
    LossArgs p, double* __restrict__ partial)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum[kStats] = {};
    for (long i = (long)blockIdx.x * 4 + wave; i < p.rows;
         i += (long)gridDim.x * 4) {
        const float m = p.mask ? p.mask[i] : 1.f;
        if (m == 0.f) continue;
        const Row r = wave_row<T>(p, i, m, lane);
        const double md = m;
        sum[0] -= md * r.surrogate;
        sum[1] += md * r.kl;
        sum[2] += md * r.entropy;
        sum[3] += md * r.escale * r.entropy;
        sum[4] += r.clipped;
        sum[5] += md;
    }
    __shared__ double s[4][kStats];
    if (lane == 0)
        for (int k = 0; k < kStats; ++k) s[wave][k] = sum[k];
    __syncthreads();
    if (threadIdx.x < kStats)
        partial[(long)blockIdx.x * kStats + threadIdx.x] =
            s[0][threadIdx.x] + s[1][threadIdx.x] + s[2][threadIdx.x] + s[3][threadIdx.x];
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
        loss[0] = (float)(s[0][0] + (double)beta * s[0][1] - (double)gamma * s[0][3]);
}

template <typename T>
__global__ __launch_bounds__(256) void policy_loss_bwd_kernel(
    LossArgs p, const float* __restrict__ upstream, T* __restrict__ grad)
{
    const int lane = threadIdx.x & 63;
    const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= p.rows) return;
    const float m = p.mask ? p.mask[i] : 1.f;
    T* out = grad + i * p.width;
    if (m == 0.f) {
        for (int j = lane; j < p.width; j += 64) store_from(out + j, 0.f);
        return;
    }
    const float g = upstream[0];
    const Row r = wave_row<T>(p, i, m, lane);
    const T* row = (const T*)p.logits + i * p.stride;
    const long a = p.action[i];
    for (int j = lane; j < p.width; j += 64)
        store_from(out + j, g * row_grad(r, load_as_float(row + j), j == a));
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
    LossArgs p;
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
        const c10::DeviceGuard guard(logits.device());
        auto stream = at::cuda::getCurrentCUDAStream();
        auto flat = logits.reshape({-1, logits.size(-1)});
        if (flat.size(1) > 1 && flat.stride(1) != 1) flat = flat.contiguous();
        const LossArgs p = make_args(flat, action, old_lp, adv, mask, escale, lo, hi, beta, gamma);
        auto fp32 = logits.options().dtype(torch::kFloat32);
        auto loss = torch::empty({}, fp32);
        auto stats = torch::empty({kStats}, fp32);
        const int blocks = (int)std::min<long>((p.rows + 3) / 4, 1024);
        auto partial = torch::empty({blocks, kStats}, fp32.dtype(torch::kFloat64));
        if (blocks > 0) {
            if (logits.scalar_type() == torch::kBFloat16)
                hipLaunchKernelGGL(policy_loss_fwd_kernel<__hip_bfloat16>, dim3(blocks),
                    dim3(256), 0, stream, p, partial.data_ptr<double>());
            else
                hipLaunchKernelGGL(policy_loss_fwd_kernel<float>, dim3(blocks),
                    dim3(256), 0, stream, p, partial.data_ptr<double>());
        }
        hipLaunchKernelGGL(policy_loss_finish_kernel, dim3(1), dim3(256), 0, stream,
            partial.data_ptr<double>(), blocks, p.beta, p.gamma,
            loss.data_ptr<float>(), stats.data_ptr<float>());
        C10_HIP_KERNEL_LAUNCH_CHECK();
        ctx->save_for_backward({logits, action, old_lp, adv, mask, escale});
        ctx->saved_data["coefs"] = std::vector<double>{lo, hi, beta, gamma};
        ctx->mark_non_differentiable({stats});
        return {loss, stats};
    }

    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        TORCH_CHECK(!at::GradMode::is_enabled(),
                    "clipped_policy_loss: its gradient is not differentiable again");
        auto saved = ctx->get_saved_variables();
        auto logits = saved[0];
        const auto coefs = ctx->saved_data["coefs"].toDoubleVector();
        const c10::DeviceGuard guard(logits.device());
        auto stream = at::cuda::getCurrentCUDAStream();
        auto flat = logits.reshape({-1, logits.size(-1)});
        if (flat.size(1) > 1 && flat.stride(1) != 1) flat = flat.contiguous();
        const LossArgs p = make_args(flat, saved[1], saved[2], saved[3], saved[4], saved[5],
                                     coefs[0], coefs[1], coefs[2], coefs[3]);
        auto grad = torch::empty(logits.sizes(), logits.options());
        auto up = grads[0].to(torch::kFloat32);
        const long blocks = (p.rows + 3) / 4;
        if (blocks > 0) {
            if (logits.scalar_type() == torch::kBFloat16)
                hipLaunchKernelGGL(policy_loss_bwd_kernel<__hip_bfloat16>, dim3(blocks),
                    dim3(256), 0, stream, p, up.data_ptr<float>(),
                    (__hip_bfloat16*)grad.data_ptr());
            else
                hipLaunchKernelGGL(policy_loss_bwd_kernel<float>, dim3(blocks), dim3(256), 0,
                    stream, p, up.data_ptr<float>(), (float*)grad.data_ptr());
            C10_HIP_KERNEL_LAUNCH_CHECK();
        }
        torch::autograd::variable_list out(10);
        out[0] = grad;
        return out;
    }
};

std::vector<torch::Tensor> clipped_policy_loss(
    const torch::Tensor& logits, const torch::Tensor& action, const torch::Tensor& old_lp,
    const torch::Tensor& adv, const c10::optional<torch::Tensor>& mask,
    const c10::optional<torch::Tensor>& escale, double lo, double hi, double beta, double gamma)
{
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
    return PolicyLoss::apply(
        logits, per_row(action, "actions", rows, logits, torch::kLong),
        per_row(old_lp, "old_log_probs", rows, logits, torch::kFloat32),
        per_row(adv, "advantages", rows, logits, torch::kFloat32),
        maybe(mask, "mask"), maybe(escale, "entropy_scale"),
        lo, hi, beta, gamma);
}

}  // namespace

void bind_policy_loss(pybind11::module& m)
{
    m.def("clipped_policy_loss", &clipped_policy_loss,
          "clipped policy loss with KL term and entropy bonus (loss, stats)");
}
