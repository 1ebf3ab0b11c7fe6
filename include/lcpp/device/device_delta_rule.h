/*
 * DeviceDeltaRule — the gated delta rule over sequences with its backward pass
 * and single-token step, through lcpp_delta_rule_*() of liblcpp_b200.so (see
 * lcpp_b200.h for the formulas).  No counterpart in the reference; calls are
 * recorded and committed like those of the other classes.
 *
 * Element types: float, __half, __nv_bfloat16; decays, strengths and states are
 * float.  Matrices are [rows][heads][dimension] in the BufferViews given, without
 * gaps.  BufferViews that may be left out are empty ones.
 */
#pragma once
#include "lcpp/device/device_linear_recurrence.h"

namespace luisa::parallel_primitive {

// Heads of queries and keys (key_heads divides heads) and of values, and their dimensions (up to 128).
struct DeltaHeads {
    uint heads = 1, key_heads = 1, key_dim = 64, value_dim = 64;
    size_t keys() const { return (size_t)key_heads * key_dim; }
    size_t values() const { return (size_t)heads * value_dim; }
    size_t state() const { return values() * key_dim; }
};

class DeviceDeltaRule : public LuisaModule {
  public:
    void create(Device& device, Stream* debug_stream = nullptr) {
        m_device = device;
        m_debug_stream = debug_stream;
    }

    // For Forward, or (backward) for both calls, with so many rows and sequences or fewer.
    template <SequenceFloatT T>
    static size_t GetTempStorageBytes(size_t num_rows, size_t num_sequences, DeltaHeads heads, bool backward = true) {
        const lcpp_delta_shape shape = of(num_rows, Sequences::of_length(num_sequences, 0), heads, 0);
        return lcpp_delta_rule_temp_bytes(lcpp_float_dtype_of<T>(), &shape, backward);
    }
    // Bytes of d_saved, which Forward fills for Backward; for so many rows and sequences or fewer.
    static size_t GetSavedStateBytes(size_t num_rows, size_t num_sequences, DeltaHeads heads) {
        const lcpp_delta_shape shape = of(num_rows, Sequences::of_length(num_sequences, 0), heads, 0);
        return lcpp_delta_rule_saved_bytes(&shape);
    }

    template <SequenceFloatT T>
    void Forward(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<T> d_q, BufferView<T> d_k, BufferView<T> d_v,
                 BufferView<float> d_decay, BufferView<float> d_beta, BufferView<T> d_out, size_t num_rows, DeltaHeads heads,
                 Sequences sequences, float scale, BufferView<float> d_init = {}, BufferView<float> d_last = {},
                 BufferView<uint> d_saved = {}) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (!inputs_fit(num_rows, heads, d_q, d_k, d_v, d_decay, d_beta) || !whole(sequences) ||
                d_out.size() < num_rows * heads.values() || !states(d_init, sequences, heads) || !states(d_last, sequences, heads) ||
                (d_saved.data() && d_saved.size_bytes() < GetSavedStateBytes(num_rows, sequences.count, heads)))
                return LCPP_ERR_INVALID_ARG;
            const lcpp_delta_shape shape = of(num_rows, sequences, heads, scale);
            const lcpp_delta_inputs in = inputs(heads, d_q, d_k, d_v, d_decay, d_beta, d_init);
            return lcpp_delta_rule_forward(lcpp_float_dtype_of<T>(), &shape, &in, d_out.data(), heads.values(), d_last.data(),
                                           d_saved.data(), temp_storage.data(), temp_storage.size_bytes(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

    // Gradients of d_q, d_k, d_v, d_decay (may be left out), d_beta and d_init (may be left out) from those of d_out and
    // of the last states (either may be left out).
    template <SequenceFloatT T>
    void Backward(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<T> d_q, BufferView<T> d_k, BufferView<T> d_v,
                  BufferView<float> d_decay, BufferView<float> d_beta, BufferView<uint> d_saved, BufferView<T> d_grad_out,
                  BufferView<T> d_grad_q, BufferView<T> d_grad_k, BufferView<T> d_grad_v, BufferView<float> d_grad_decay,
                  BufferView<float> d_grad_beta, size_t num_rows, DeltaHeads heads, Sequences sequences, float scale,
                  BufferView<float> d_init = {}, BufferView<float> d_grad_last = {}, BufferView<float> d_grad_init = {}) {
        cmdlist << [=](cudaStream_t s) -> int {
            const size_t gates = num_rows * heads.heads;
            if (!inputs_fit(num_rows, heads, d_q, d_k, d_v, d_decay, d_beta) || !whole(sequences) ||
                d_saved.size_bytes() < GetSavedStateBytes(num_rows, sequences.count, heads) ||
                (d_grad_out.data() && d_grad_out.size() < num_rows * heads.values()) || d_grad_q.size() < num_rows * heads.keys() ||
                d_grad_k.size() < num_rows * heads.keys() || d_grad_v.size() < num_rows * heads.values() ||
                (d_grad_decay.data() && d_grad_decay.size() < gates) || d_grad_beta.size() < gates ||
                !states(d_init, sequences, heads) || !states(d_grad_last, sequences, heads) || !states(d_grad_init, sequences, heads))
                return LCPP_ERR_INVALID_ARG;
            const lcpp_delta_shape shape = of(num_rows, sequences, heads, scale);
            const lcpp_delta_inputs in = inputs(heads, d_q, d_k, d_v, d_decay, d_beta, d_init);
            const lcpp_delta_grads grads{d_grad_out.data(), heads.values(), d_grad_last.data(), d_grad_q.data(), d_grad_k.data(),
                                         d_grad_v.data(), d_grad_decay.data(), d_grad_beta.data(), d_grad_init.data()};
            return lcpp_delta_rule_backward(lcpp_float_dtype_of<T>(), &shape, &in, d_saved.data(), &grads, temp_storage.data(),
                                            temp_storage.size_bytes(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

    // One token a row: row i goes on from state d_parents[i] (without parents i; a negative parent from zeros).
    template <SequenceFloatT T>
    void Step(CommandList& cmdlist, BufferView<T> d_q, BufferView<T> d_k, BufferView<T> d_v, BufferView<float> d_decay,
              BufferView<float> d_beta, BufferView<float> d_states_in, BufferView<float> d_states_out, BufferView<T> d_out,
              size_t num_rows, DeltaHeads heads, float scale, BufferView<int32_t> d_parents = {}) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (!inputs_fit(num_rows, heads, d_q, d_k, d_v, d_decay, d_beta) || d_out.size() < num_rows * heads.values() ||
                d_states_out.size() < num_rows * heads.state() || (d_parents.data() && d_parents.size() < num_rows))
                return LCPP_ERR_INVALID_ARG;
            const lcpp_delta_shape shape = of(num_rows, {}, heads, scale);
            const lcpp_delta_inputs in = inputs(heads, d_q, d_k, d_v, d_decay, d_beta, d_states_in);
            return lcpp_delta_rule_step(lcpp_float_dtype_of<T>(), &shape, &in, heads.state() ? d_states_in.size() / heads.state() : 0,
                                        d_parents.data(), d_states_out.data(), d_out.data(), heads.values(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

  private:
    static lcpp_delta_shape of(size_t rows, const Sequences& q, DeltaHeads h, float scale) {
        return {rows, q.count, q.length, q.offsets.data(), h.heads, h.key_heads, h.key_dim, h.value_dim, scale};
    }
    template <typename T>
    static bool inputs_fit(size_t rows, DeltaHeads h, BufferView<T> q, BufferView<T> k, BufferView<T> v, BufferView<float> decay,
                           BufferView<float> beta) {
        return q.size() >= rows * h.keys() && k.size() >= rows * h.keys() && v.size() >= rows * h.values() &&
               beta.size() >= rows * h.heads && (!decay.data() || decay.size() >= rows * h.heads);
    }
    template <typename T>
    static lcpp_delta_inputs inputs(DeltaHeads h, BufferView<T> q, BufferView<T> k, BufferView<T> v, BufferView<float> decay,
                                    BufferView<float> beta, BufferView<float> init) {
        return {q.data(), k.data(), v.data(), h.keys(), h.keys(), h.values(), decay.data(), beta.data(), h.heads, h.heads, init.data()};
    }
    static bool whole(const Sequences& sequences) {
        return !sequences.offsets.data() || sequences.offsets.size() > sequences.count;
    }
    static bool states(BufferView<float> v, const Sequences& sequences, DeltaHeads h) {
        return !v.data() || v.size() >= sequences.count * h.state();
    }
    Device m_device;
    Stream* m_debug_stream = nullptr;
};

}  // namespace luisa::parallel_primitive
