/*
 * DeviceCrossEntropy — softmax cross entropy over a vocabulary from hidden
 * states, without the logits in memory, and its gradients, through
 * lcpp_cross_entropy_*() of liblcpp_b200.so (see lcpp_b200.h for the formulas).
 * No counterpart in the reference; calls are recorded and committed like those
 * of the other classes.  Element types: float, __half, __nv_bfloat16.
 */
#pragma once
#include "lcpp/device/device_linear_recurrence.h"

namespace luisa::parallel_primitive {

class DeviceCrossEntropy : public LuisaModule {
  public:
    void create(Device& device, Stream* debug_stream = nullptr) {
        m_device = device;
        m_debug_stream = debug_stream;
    }

    // For Forward, or (backward) for both calls, with so many rows or fewer; aligned false: d_weight may start off a
    // 16-byte boundary.
    template <SequenceFloatT T>
    static size_t GetTempStorageBytes(size_t num_rows, size_t num_channels, size_t vocab, bool backward = true, bool aligned = true) {
        return lcpp_cross_entropy_temp_bytes(lcpp_float_dtype_of<T>(), num_rows, num_channels, vocab, backward, aligned);
    }

    // d_hidden [rows][channels], d_weight [vocab][channels], d_targets [rows] (negative: the row takes no part); d_loss and
    // d_logsum (for Backward) [rows], either may be left out.
    template <SequenceFloatT T>
    void Forward(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<T> d_hidden, BufferView<T> d_weight,
                 BufferView<int32_t> d_targets, BufferView<float> d_loss, BufferView<float> d_logsum, size_t num_rows,
                 size_t num_channels, size_t vocab) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (!fit(d_hidden, d_weight, d_targets, num_rows, num_channels, vocab) || (d_loss.data() && d_loss.size() < num_rows) ||
                (d_logsum.data() && d_logsum.size() < num_rows))
                return LCPP_ERR_INVALID_ARG;
            return lcpp_cross_entropy_forward(lcpp_float_dtype_of<T>(), d_hidden.data(), num_channels, d_weight.data(), num_channels,
                                              d_targets.data(), d_loss.data(), d_logsum.data(), num_rows, num_channels, vocab,
                                              temp_storage.data(), temp_storage.size_bytes(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

    // d_grad_loss: one value for each row, or a single one for all; d_grad_hidden and d_grad_weight: either may be left out.
    template <SequenceFloatT T>
    void Backward(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<T> d_hidden, BufferView<T> d_weight,
                  BufferView<int32_t> d_targets, BufferView<float> d_logsum, BufferView<float> d_grad_loss,
                  BufferView<T> d_grad_hidden, BufferView<T> d_grad_weight, size_t num_rows, size_t num_channels, size_t vocab) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (!fit(d_hidden, d_weight, d_targets, num_rows, num_channels, vocab) || d_logsum.size() < num_rows ||
                (d_grad_loss.size() < num_rows && d_grad_loss.size() != 1) ||
                (d_grad_hidden.data() && d_grad_hidden.size() < num_rows * num_channels) ||
                (d_grad_weight.data() && d_grad_weight.size() < vocab * num_channels))
                return LCPP_ERR_INVALID_ARG;
            return lcpp_cross_entropy_backward(lcpp_float_dtype_of<T>(), d_hidden.data(), num_channels, d_weight.data(), num_channels,
                                               d_targets.data(), d_logsum.data(), d_grad_loss.data(),
                                               d_grad_loss.size() == 1 ? 0 : 1, d_grad_hidden.data(), num_channels,
                                               d_grad_weight.data(), num_channels, num_rows, num_channels, vocab,
                                               temp_storage.data(), temp_storage.size_bytes(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

  private:
    template <typename T>
    static bool fit(BufferView<T> hidden, BufferView<T> weight, BufferView<int32_t> targets, size_t rows, size_t channels, size_t vocab) {
        return hidden.size() >= rows * channels && weight.size() >= vocab * channels && targets.size() >= rows;
    }
    Device m_device;
    Stream* m_debug_stream = nullptr;
};

}  // namespace luisa::parallel_primitive
