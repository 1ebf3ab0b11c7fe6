/*
 * DeviceBeamSearch — selection of the best continuations over beams and
 * vocabulary, and states that follow their beams, through lcpp_beam_select() /
 * lcpp_beam_reorder() of liblcpp_b200.so (see lcpp_b200.h).  No counterpart in
 * the reference; calls are recorded and committed like those of the other
 * classes.  Logits: float, __half or __nv_bfloat16, [batches * beams][vocab].
 */
#pragma once
#include "lcpp/device/device_linear_recurrence.h"

namespace luisa::parallel_primitive {

class DeviceBeamSearch : public LuisaModule {
  public:
    void create(Device& device, Stream* debug_stream = nullptr) {
        m_device = device;
        m_debug_stream = debug_stream;
    }

    static size_t GetTempStorageBytes(size_t num_batches, uint num_beams, size_t vocab) {
        return lcpp_beam_select_temp_bytes(num_batches, num_beams, vocab);
    }

    // The `num_beams` best continuations of every batch entry, best first: score, token, parent (a row of d_logits)
    // and whether it is finished.  d_finished_in and d_finished_out may be empty; eos_token < 0: there is none.
    template <SequenceFloatT T>
    void Select(CommandList& cmdlist, BufferView<uint> temp_storage, BufferView<T> d_logits, BufferView<float> d_scores_in,
                BufferView<uint8_t> d_finished_in, BufferView<float> d_scores_out, BufferView<int32_t> d_tokens_out,
                BufferView<int32_t> d_parents_out, BufferView<uint8_t> d_finished_out, size_t num_batches,
                uint num_beams, size_t vocab, int32_t eos_token = -1) {
        cmdlist << [=](cudaStream_t s) -> int {
            const size_t rows = num_batches * num_beams;
            if (d_logits.size() < rows * vocab || d_scores_in.size() < rows || d_scores_out.size() < rows ||
                d_tokens_out.size() < rows || d_parents_out.size() < rows ||
                (d_finished_in.data() && d_finished_in.size() < rows) ||
                (d_finished_out.data() && d_finished_out.size() < rows))
                return LCPP_ERR_INVALID_ARG;
            return lcpp_beam_select(lcpp_float_dtype_of<T>(), d_logits.data(), vocab, d_scores_in.data(),
                                    d_finished_in.data(), d_scores_out.data(), d_tokens_out.data(), d_parents_out.data(),
                                    d_finished_out.data(), num_batches, num_beams, vocab, eos_token, temp_storage.data(),
                                    temp_storage.size_bytes(), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

    // d_out[l][i] = d_in[l][d_parents[i]] for [layers][rows][width] states of any element type.
    template <typename T>
    void Reorder(CommandList& cmdlist, BufferView<T> d_in, BufferView<T> d_out, BufferView<int32_t> d_parents,
                 size_t num_layers, size_t rows_in, size_t rows, size_t width) {
        cmdlist << [=](cudaStream_t s) -> int {
            if (d_in.size() < num_layers * rows_in * width || d_out.size() < num_layers * rows * width ||
                d_parents.size() < rows)
                return LCPP_ERR_INVALID_ARG;
            return lcpp_beam_reorder(d_in.data(), rows_in * width * sizeof(T), width * sizeof(T), d_out.data(),
                                     rows * width * sizeof(T), width * sizeof(T), d_parents.data(), num_layers, rows_in,
                                     rows, width * sizeof(T), s);
        };
        lcpp_check(cmdlist, m_debug_stream);
    }

  private:
    Device m_device;
    Stream* m_debug_stream = nullptr;
};

}  // namespace luisa::parallel_primitive
