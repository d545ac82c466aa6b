// Refusals that the operators with gradients share (guards.hip).
#pragma once

#include <torch/extension.h>

// The kernels give no forward-mode derivatives; a result without one would count
// as constant.
void check_forward_mode(const char* op, std::initializer_list<c10::optional<torch::Tensor>> all);

// The capture that the current stream is in, or 0.
int64_t capture_now();

// For a backward pass, whose forward pass was in the capture `then` (0: in none).
void check_capture(const char* op, int64_t then);
