// dnn/optimizers/adamw_optimizer.hpp -- AdamW for the C++ drop-in.
//
// The reference has Adam with coupled decay only
// (dnn/optimizers/adam_optimizer.cu:83-130); this optimizer keeps its interface
// (dnn/optimizers/optimizer.cuh) with the decay decoupled from the moments.
// Provided for T = float, the element type of the Linear layer's weight and
// bias gradients; one df_adamw_update call updates the whole list.
//
// state_bits 32: the moments in binary32; 8: as e4m3 codes with a scale per 256
// values, dithered (a quarter of the memory; see df_adamw_update_dithered in
// include/df_capi.h).  A parameter is known
// by its tensor's address, its moments start at zero when update_parameters
// first lists it, or lists it with another size; step() refuses one whose size
// changed after that (tensor::load gives a tensor another shape and buffer).
// set_weight_decay(param, wd) gives one parameter a decay of its own (0 for
// biases and norms, usually).  step_clipped(max_norm) is step() on gradients
// clipped to that global norm, which keep their values.
#pragma once

#include <memory>
#include <unordered_map>

#include "dnn/optimizers/optimizer.hpp"

namespace dnn {

template <typename T>
class AdamWOptimizer : public Optimizer<T> {
public:
    AdamWOptimizer(T learning_rate = 0.001, T beta1 = 0.9, T beta2 = 0.999, T epsilon = 1e-8, T weight_decay = 0.01,
                   int state_bits = 32);

    void step() override;
    void zero_grad() override;
    void update_parameters(const std::vector<tensor<T>*>& parameters,
                           const std::vector<tensor<T>*>& gradients) override;

    T learning_rate() const override { return learning_rate_; }
    void set_learning_rate(T new_lr) override { learning_rate_ = new_lr; }
    void set_weight_decay(const tensor<T>* param, T weight_decay) { decay_[param] = weight_decay; }

    const float* step_clipped(float max_norm);  // the norm, on the device
    int timestep() const { return timestep_; }
    int state_bits() const { return state_bits_; }

private:
    struct State {
        std::unique_ptr<tensor<T>> m, v;                // 32 bits
        std::unique_ptr<tensor<uint8_t>> mq, vq;        // 8 bits: codes
        std::unique_ptr<tensor<float>> m_scale, v_scale;
        int64_t size() const { return m ? m->size() : mq->size(); }
    };
    void launch(const float* clip_norm, float max_norm);

    T learning_rate_, beta1_, beta2_, epsilon_, weight_decay_;
    int state_bits_, timestep_ = 0;
    std::unordered_map<const tensor<T>*, State> state_;
    std::unordered_map<const tensor<T>*, T> decay_;
};

}  // namespace dnn
