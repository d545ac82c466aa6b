#include "guards.h"

#include <torch/csrc/autograd/function.h>
#include <ATen/cuda/CUDAContext.h>
#include <hip/hip_runtime.h>

void check_forward_mode(const char* op, std::initializer_list<c10::optional<torch::Tensor>> all)
{
    for (auto& t : all)
        TORCH_CHECK_VALUE(!t || !t->_fw_grad(0).defined(), op,
                          ": has no forward-mode derivative on the GPU");
}

int64_t capture_now()
{
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    C10_HIP_CHECK(hipStreamGetCaptureInfo(at::cuda::getCurrentCUDAStream(), &status, &id));
    return status == hipStreamCaptureStatusActive ? (int64_t)id : 0;
}

// A captured backward pass of an eager forward pass would draw the leaves' own
// streams into the capture, which never join it.  Where a gradient goes to a node
// that an eager graph made on the default stream and keeps alive, torch lets that
// stream wait for this one: it cannot be drawn into a capture, and the process
// ends there.
void check_capture(const char* op, int64_t then)
{
    if (capture_now() == 0) return;
    TORCH_CHECK(then != 0, op, ": a captured backward pass needs a captured forward pass");
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        const auto& to = node->next_edge(i).function;
        if (!to || !node->task_should_compute_output(i)) continue;
        const auto stream = to->stream();
        TORCH_CHECK(!stream ||
                    stream->id() != at::cuda::getDefaultCUDAStream(stream->device_index()).id(),
                    op, ": a captured backward pass needs inputs without a living eager graph: "
                    "what eager passes over them returned has to be gone");
    }
}
