/*
 * DeviceLinearRecurrence — gated linear recurrences over sequences with their
 * backward pass and single-token step, through lcpp_linear_recurrence_*() of
 * liblcpp_b200.so (see lcpp_b200.h for the formulas).  No counterpart in the
 * reference; calls are recorded and committed like those of the other classes.
 *
 * Element types: float, __half, __nv_bfloat16; states are float.  Matrices are
 * [rows][channels] in the BufferViews given; `sequences` describes how the rows
 * are divided.  BufferViews that may be left out are empty ones.
 */
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "lcpp/runtime/core.h"

namespace luisa::parallel_primitive {

// Element type -> lcpp_dtype of the sequence operators.
template <typename T>
constexpr int lcpp_float_dtype_of() {
    if constexpr (std::is_same_v<T, float>) return LCPP_F32;
    else if constexpr (std::is_same_v<T, __half>) return LCPP_F16;
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return LCPP_BF16;
    else return -1;
}
template <typename T>
concept SequenceFloatT = lcpp_float_dtype_of<T>() >= 0;

// h = gate h' + in; the product of the gates along up to 128 rows must stay finite
struct LinearGate { static constexpr int lcpp_gate = LCPP_GATE_LINEAR; };
struct SigmoidGate { static constexpr int lcpp_gate = LCPP_GATE_SIGMOID; };  // h = a h' + (1 - a) in, a = sigmoid(gate)

// Rows of equal sequences, or CSR row offsets (num_sequences + 1 on the device).
struct Sequences {
    size_t count = 0, length = 0;
    luisa::compute::BufferView<luisa::uint> offsets;
    static Sequences of_length(size_t count, size_t length) { return {count, length, {}}; }
    static Sequences of_offsets(luisa::compute::BufferView<luisa::uint> offsets) {
        return {offsets.size() ? offsets.size() - 1 : 0, 0, offsets};
    }
};

class DeviceLinearRecurrence : public LuisaModule {
  public:
    void create(Device& device, Stream* debug_stream = nullptr) {
        m_device = device;
        m_debug_stream = debug_stream;
    }

    static size_t GetTempStorageBytes(size_t num_rows, size_t num_channels) {
        return lcpp_linear_recurrence_temp_bytes(num_rows, num_channels);
    }
    // Bytes of d_saved, which Forward fills for Backward.
    static size_t GetSavedStateBytes(size_t num_rows, size_t num_channels) {
        return lcpp_linear_recurrence_saved_bytes(num_rows, num_channels);
    }

    template <typename Gate, SequenceFloatT T>
    void Forward(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<T> d_gate, BufferView<T> d_in,
                 BufferView<T> d_out, size_t num_rows, size_t num_channels, Sequences sequences, Gate,
                 BufferView<float> d_init = {}, BufferView<float> d_last = {}, BufferView<uint> d_saved = {}) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (!whole(sequences) || !fits(d_gate, num_rows, num_channels) || !fits(d_in, num_rows, num_channels) ||
                !fits(d_out, num_rows, num_channels) || !states(d_init, sequences, num_channels) ||
                !states(d_last, sequences, num_channels) || !saved(d_saved, num_rows, num_channels))
                return LCPP_ERR_INVALID_ARG;
            return lcpp_linear_recurrence_forward(Gate::lcpp_gate, lcpp_float_dtype_of<T>(), d_gate.data(), num_channels,
                                                  d_in.data(), num_channels, d_out.data(), num_channels, num_rows,
                                                  num_channels, sequences.count, sequences.length,
                                                  sequences.offsets.data(), d_init.data(), num_channels, d_last.data(),
                                                  d_saved.data(), temp_storage.data(), temp_storage.size_bytes(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

    template <typename Gate, SequenceFloatT T>
    void Backward(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<T> d_gate, BufferView<T> d_in,
                  BufferView<uint> d_saved, BufferView<T> d_grad_out, BufferView<T> d_grad_gate,
                  BufferView<T> d_grad_in, size_t num_rows, size_t num_channels, Sequences sequences, Gate,
                  BufferView<float> d_init = {}, BufferView<float> d_grad_last = {},
                  BufferView<float> d_grad_init = {}) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (!whole(sequences) || !fits(d_gate, num_rows, num_channels) || !fits(d_in, num_rows, num_channels) ||
                !fits(d_grad_gate, num_rows, num_channels) || !fits(d_grad_in, num_rows, num_channels) ||
                (d_grad_out.data() && !fits(d_grad_out, num_rows, num_channels)) ||
                !states(d_init, sequences, num_channels) || !states(d_grad_last, sequences, num_channels) ||
                !states(d_grad_init, sequences, num_channels) || !saved(d_saved, num_rows, num_channels))
                return LCPP_ERR_INVALID_ARG;
            return lcpp_linear_recurrence_backward(
                Gate::lcpp_gate, lcpp_float_dtype_of<T>(), d_gate.data(), num_channels, d_in.data(), num_channels,
                d_saved.data(), d_init.data(), num_channels, d_grad_out.data(), num_channels, d_grad_last.data(),
                d_grad_gate.data(), num_channels, d_grad_in.data(), num_channels, d_grad_init.data(), num_rows,
                num_channels, sequences.count, sequences.length, sequences.offsets.data(), temp_storage.data(),
                temp_storage.size_bytes(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

    // One token a row: row i goes on from state d_parents[i] (without parents i; a negative parent from zeros).
    template <typename Gate, SequenceFloatT T>
    void Step(CommandList& cmdlist, BufferView<T> d_gate, BufferView<T> d_in, BufferView<float> d_states_in,
              BufferView<float> d_states_out, BufferView<T> d_out, size_t num_rows, size_t num_channels, Gate,
              BufferView<int32_t> d_parents = {}) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (!fits(d_gate, num_rows, num_channels) || !fits(d_in, num_rows, num_channels) ||
                !fits(d_states_out, num_rows, num_channels) || (d_out.data() && !fits(d_out, num_rows, num_channels)) ||
                (d_parents.data() && d_parents.size() < num_rows))
                return LCPP_ERR_INVALID_ARG;
            return lcpp_linear_recurrence_step(Gate::lcpp_gate, lcpp_float_dtype_of<T>(), d_gate.data(), num_channels,
                                               d_in.data(), num_channels, d_states_in.data(),
                                               num_channels ? d_states_in.size() / num_channels : 0, d_parents.data(),
                                               d_states_out.data(), d_out.data(), num_channels, num_rows, num_channels, s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

  private:
    template <typename T>
    static bool fits(BufferView<T> m, size_t rows, size_t channels) { return m.size() >= rows * channels; }
    static bool whole(const Sequences& sequences) {
        return !sequences.offsets.data() || sequences.offsets.size() > sequences.count;
    }
    static bool states(BufferView<float> v, const Sequences& sequences, size_t channels) {
        return !v.data() || v.size() >= sequences.count * channels;
    }
    static bool saved(BufferView<uint> v, size_t rows, size_t channels) {
        return !v.data() || v.size_bytes() >= GetSavedStateBytes(rows, channels);
    }
    Device m_device;
    Stream* m_debug_stream = nullptr;
};

}  // namespace luisa::parallel_primitive
