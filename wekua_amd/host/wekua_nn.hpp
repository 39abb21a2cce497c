// wekua_nn.hpp -- host-side mirror of the part of wekua's `nn` / `math` modules that one MLP
// training step uses, on top of wekua.hpp and the C ABI (include/wekua_hip.h):
//
//   wekua::math::dot / sum / mean       src/math/basic.zig:18-77,128-244
//   wekua::nn::Activation, Sigmoid, Tanh  src/nn/activation/{main,sigmoid,tanh}.zig
//   wekua::nn::Layer (interface)        src/nn/layer/main.zig:14-135
//   wekua::nn::Linear                   src/nn/layer/linear.zig
//   wekua::nn::Sequential               src/nn/layer/sequential.zig
//   wekua::nn::Cache                    src/nn/layer/cache.zig
//   wekua::nn::loss::mse                src/nn/loss/mse.zig:63-132
//   wekua::nn::optimizers::GD           src/nn/optimizers/gd.zig (w += -lr * g through blas.axpy)
//   wekua::nn::Identity, Dropout, TokenLogProbs, loss::tokens  no Zig counterpart: what training on tokens
//                                       needs around the layers above
//   wekua::nn::optimizers::Adam         no Zig counterpart (src/nn/optimizers/adam.zig is empty):
//                                       textbook Adam, see wk_adam_step
//
// Differences chosen for this device: bias add and activation run as one fused kernel after the
// forward GEMM (same arithmetic, one pass over the output instead of two); the Xavier-uniform
// weight initialisation is drawn on the host and uploaded (the reference seeds its device generator
// from the wall clock, linear.zig:125-132, so there is no reproducible stream to match) and takes
// an optional seed.
#pragma once

#include <atomic>
#include <chrono>
#include <cmath>
#include <limits>
#include <memory>

#include "wekua.hpp"

namespace wekua {

namespace math {
// x = x * y element-wise, in place (math.dot)
template <typename T> void dot(Pipeline *pipeline, Tensor<T> *x, Tensor<T> *y) {
    helpers::eqlTensorsShape<T>(x, y);
    const uint64_t shape3[3] = {x->depth(), x->rows(), x->cols()};
    check(wk_hadamard(pipeline->command_queue->stream, core::getTypeIndex<T>(), shape3, x->buffer, x->memory_layout.row_pitch,
                      x->memory_layout.slice_pitch, y->buffer, y->memory_layout.row_pitch, y->memory_layout.slice_pitch));
    pipeline->append(1);
}

// scale * sum of all logical elements, returned on the host (synchronises the pipeline, as
// math.sum / math.mean do: src/math/basic.zig:128-244)
template <typename T> T scaledSum(Pipeline *pipeline, Tensor<T> *x, double scale) {
    const Context *ctx = x->context;
    void *ws = nullptr, *res = nullptr;
    check(wk_malloc(ctx->device, wk_sum_workspace_bytes(core::getTypeIndex<T>()), &ws));
    int rc = wk_malloc(ctx->device, sizeof(T), &res);
    if (rc) {
        wk_free(ctx->device, ws);
        throw Error(rc);
    }
    const uint64_t shape3[3] = {x->depth(), x->rows(), x->cols()};
    T host = T(0);
    rc = wk_sum(pipeline->command_queue->stream, core::getTypeIndex<T>(), shape3, x->buffer, x->memory_layout.row_pitch,
                x->memory_layout.slice_pitch, ws, res, scale);
    if (!rc)
        rc = wk_copy_d2h_rect_async(pipeline->command_queue->stream, &host, sizeof(T), 0, res, sizeof(T), 0, sizeof(T), 1, 1);
    if (!rc) {
        pipeline->append(1);
        pipeline->waitAndCleanup();
    }
    wk_free(ctx->device, ws);
    wk_free(ctx->device, res);
    check(rc);
    return host;
}
template <typename T> T sum(Pipeline *pipeline, Tensor<T> *x) { return scaledSum<T>(pipeline, x, 1.0); }
template <typename T> T mean(Pipeline *pipeline, Tensor<T> *x) {
    return scaledSum<T>(pipeline, x, 1.0 / (double)x->dimensions.number_of_elements_without_padding);
}
} // namespace math

namespace nn {

// ---- activations ----------------------------------------------------------------------------
// No counterpart in the reference, whose layers without an activation get zero gradients: the derivative is one.  The
// activation of a last layer whose outputs are logits.
constexpr int IDENTITY = 2;

template <typename T> struct Activation {
    int kind = WK_ACT_NONE;
    // in place on the layer output (Activation.run)
    void run(Pipeline *pipeline, Tensor<T> *net_output) const {
        if (kind == IDENTITY) return;
        const uint64_t shape3[3] = {net_output->depth(), net_output->rows(), net_output->cols()};
        check(wk_activation(pipeline->command_queue->stream, core::getTypeIndex<T>(), kind, shape3, net_output->buffer,
                            net_output->memory_layout.row_pitch, net_output->memory_layout.slice_pitch));
        pipeline->append(1);
    }
    // derivative expressed through the activation output (Activation.getDerivative)
    void getDerivative(Pipeline *pipeline, Tensor<T> *output, Tensor<T> *derivative) const {
        helpers::eqlTensorsShape<T>(output, derivative);
        if (kind == IDENTITY) return fill::one<T>(pipeline, derivative);
        const uint64_t shape3[3] = {output->depth(), output->rows(), output->cols()};
        check(wk_activation_dev(pipeline->command_queue->stream, core::getTypeIndex<T>(), kind, shape3, output->buffer,
                                output->memory_layout.row_pitch, output->memory_layout.slice_pitch, derivative->buffer,
                                derivative->memory_layout.row_pitch, derivative->memory_layout.slice_pitch));
        pipeline->append(1);
    }
};
template <typename T> struct Sigmoid {
    static Activation<T> init() { return Activation<T>{WK_ACT_SIGMOID}; }
};
template <typename T> struct Tanh {
    static Activation<T> init() { return Activation<T>{WK_ACT_TANH}; }
};
template <typename T> struct Identity {
    static Activation<T> init() { return Activation<T>{IDENTITY}; }
};

// ---- Layer interface (src/nn/layer/main.zig: the vtable) ---------------------------------------
template <typename T> struct Layer {
    using TensorT = Tensor<T>;
    virtual ~Layer() = default;
    virtual void deinit(Pipeline *pipeline) = 0;
    virtual TensorT *getCachedOutput(const void *cache) const = 0;
    virtual std::vector<TensorT *> getWeights() const = 0;
    virtual std::vector<TensorT *> getBias() const = 0; // entries may be null
    virtual void *prepareCache(Pipeline *pipeline, uint64_t number_of_elements) const = 0;
    virtual void releaseCache(Pipeline *pipeline, void *cache) const = 0;
    virtual TensorT *forward(Pipeline *pipeline, TensorT *input, void *cache) const = 0;
    virtual TensorT *getSensitivity(const void *cache) const = 0;
    virtual void backward(Pipeline *pipeline, void *cache, TensorT *input, TensorT *input_gradient) const = 0;
    virtual std::vector<TensorT *> getGradients(const void *cache) const = 0;
    virtual std::vector<TensorT *> getBiasGradients(const void *cache) const = 0; // entries may be null
    // no counterpart in the reference: what Dropout listens to
    virtual void setTraining(bool) {}
    virtual void setStep(Tensor<uint64_t> *) {}
};

// ---- Linear ------------------------------------------------------------------------------------
struct ExtraParams {
    size_t deep = 1;         // src/nn/layer/linear.zig:23-26: extra {output, output} layers behind the first
    bool enable_bias = true;
    // Seed of the Xavier-uniform initialisation.  The reference seeds tensor.random.uniform from the
    // clock (linear.zig:125-132: seed == null); nullopt does the same here, a value makes it repeatable.
    std::optional<uint64_t> seed = std::nullopt;
};

namespace detail {
inline uint64_t splitmix64(uint64_t &state) {
    uint64_t z = (state += 0x9E3779B97F4A7C15ull);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
// uniform in [-limit, limit), limit = sqrt(6 / (input + output))  (getRandomLimits, linear.zig:28-45)
template <typename T> void xavierUniform(Pipeline *pipeline, Tensor<T> *w, uint64_t input, uint64_t output, uint64_t &state) {
    const double limit = std::sqrt(6.0 / (double)(input + output));
    std::vector<T> host(w->dimensions.number_of_elements_without_padding);
    for (T &v : host) v = (T)((2.0 * ((double)(splitmix64(state) >> 11) * 0x1.0p-53) - 1.0) * limit);
    memory::readFromBuffer<T>(pipeline, w, host.data(), host.size());
    pipeline->waitAndCleanup(); // `host` dies with this scope
}
} // namespace detail

template <typename T> struct Linear : Layer<T> {
    using TensorT = Tensor<T>;
    struct LinearCache {
        std::vector<TensorT *> outputs, sensitivities, acti_derivatives, gradients, bias_gradients;
    };

    const Context *context = nullptr;
    std::vector<TensorT *> weights; // [0] is {output, input}, the rest {output, output}
    std::vector<TensorT *> bias;    // {output} each, or nulls when disabled
    bool bias_enabled = true;
    std::optional<Activation<T>> activation;

    // Linear.init (linear.zig:86-180)
    static Linear *init(const Context *context, Pipeline *pipeline, uint64_t input, uint64_t output,
                        std::optional<Activation<T>> acti, ExtraParams extra = {}) {
        if (input == 0 || output == 0 || extra.deep == 0) throw Error(WK_E_INVALID_VALUE);
        auto self = std::make_unique<Linear>();
        self->context = context;
        self->activation = acti;
        self->bias_enabled = extra.enable_bias;
        uint64_t state = extra.seed ? *extra.seed : (uint64_t)std::chrono::steady_clock::now().time_since_epoch().count();
        try {
            for (size_t i = 0; i < extra.deep; ++i) {
                const uint64_t in = i == 0 ? input : output;
                self->weights.push_back(TensorT::alloc(context, pipeline, {output, in}));
                detail::xavierUniform<T>(pipeline, self->weights.back(), in, output, state);
            }
            self->bias.assign(extra.deep, nullptr);
            if (extra.enable_bias)
                for (size_t i = 0; i < extra.deep; ++i) self->bias[i] = TensorT::alloc(context, pipeline, {output});
        } catch (...) {
            for (TensorT *t : self->weights) t->release(pipeline);
            for (TensorT *t : self->bias)
                if (t) t->release(pipeline);
            throw;
        }
        return self.release();
    }
    void deinit(Pipeline *pipeline) override {
        for (TensorT *t : weights) t->release(pipeline);
        for (TensorT *t : bias)
            if (t) t->release(pipeline);
        delete this;
    }
    TensorT *getCachedOutput(const void *cache) const override { return static_cast<const LinearCache *>(cache)->outputs.back(); }
    std::vector<TensorT *> getWeights() const override { return weights; }
    std::vector<TensorT *> getBias() const override { return bias; }

    // prepareCache (linear.zig:202-398): per-batch-size outputs, sensitivities (filled with one),
    // activation derivatives (zero), gradients and bias gradients
    void *prepareCache(Pipeline *pipeline, uint64_t number_of_elements) const override {
        if (number_of_elements == 0) throw Error(WK_E_INVALID_VALUE);
        auto c = std::make_unique<LinearCache>();
        try {
            for (size_t i = 0; i < weights.size(); ++i) {
                const auto &wshape = weights[i]->dimensions.shape;
                c->outputs.push_back(TensorT::alloc(context, pipeline, {number_of_elements, wshape[0]}));
                c->sensitivities.push_back(TensorT::alloc(context, pipeline, {number_of_elements, wshape[0]}));
                c->acti_derivatives.push_back(TensorT::alloc(context, pipeline, {number_of_elements, wshape[0]}));
                fill::one<T>(pipeline, c->sensitivities.back());
                c->gradients.push_back(TensorT::alloc(context, pipeline, wshape));
                c->bias_gradients.push_back(TensorT::alloc(context, pipeline, {wshape[0]}));
            }
        } catch (...) {
            releaseCache(pipeline, c.release());
            throw;
        }
        return c.release();
    }
    void releaseCache(Pipeline *pipeline, void *cache) const override {
        LinearCache *c = static_cast<LinearCache *>(cache);
        for (auto *list : {&c->outputs, &c->sensitivities, &c->acti_derivatives, &c->gradients, &c->bias_gradients})
            for (TensorT *t : *list) t->release(pipeline);
        delete c;
    }

    // forward (linear.zig:480-525): out = in * W^T, then addBias and the activation -- here one
    // call: bias and activation run in the epilogue of the matrix-core kernel
    TensorT *forward(Pipeline *pipeline, TensorT *input, void *cache) const override {
        LinearCache *c = static_cast<LinearCache *>(cache);
        for (size_t i = 0; i < weights.size(); ++i) {
            TensorT *out = c->outputs[i];
            blas::validateTensors<T>(input, weights[i], out, blas::Operation::no_transpose, blas::Operation::transpose);
            check(wk_gemm_bias_activation(pipeline->command_queue->stream, core::getTypeIndex<T>(), 0, 1, out->rows(), out->cols(),
                                          input->cols(), input->buffer, input->memory_layout.row_pitch, weights[i]->buffer,
                                          weights[i]->memory_layout.row_pitch, out->buffer, out->memory_layout.row_pitch,
                                          bias_enabled ? bias[i]->buffer : nullptr,
                                          activation && activation->kind != IDENTITY ? activation->kind : WK_ACT_NONE));
            pipeline->append(1);
            input = out;
        }
        return input;
    }
    TensorT *getSensitivity(const void *cache) const override {
        return static_cast<const LinearCache *>(cache)->sensitivities.back();
    }

    // backward (linear.zig:579-678).  As there, the sensitivity is multiplied by the cached
    // derivative tensor even when the layer has no activation; that tensor then still holds the
    // zeros it was created with, so such a layer yields zero gradients.
    void backward(Pipeline *pipeline, void *cache, TensorT *input, TensorT *input_sensitivity) const override {
        LinearCache *c = static_cast<LinearCache *>(cache);
        TensorT *sens = c->sensitivities.back();
        for (size_t i = weights.size(); i-- > 0;) {
            TensorT *prev_output = i >= 1 ? c->outputs[i - 1] : input;
            // activation derivative from the cached output, Hadamard product into the sensitivity and the
            // bias gradient (column sums of the new sensitivity) in one pass over the layer's output
            TensorT *dev = c->acti_derivatives[i];
            helpers::eqlTensorsShape<T>(sens, dev);
            helpers::eqlTensorsShape<T>(sens, c->outputs[i]);
            if (activation && activation->kind == IDENTITY) {
                if (bias_enabled) // the sensitivity stays what it is
                    check(wk_bias_step(pipeline->command_queue->stream, core::getTypeIndex<T>(), sens->rows(), sens->cols(), sens->buffer,
                                       sens->memory_layout.row_pitch, c->bias_gradients[i]->buffer));
            } else {
                check(wk_sensitivity_step(pipeline->command_queue->stream, core::getTypeIndex<T>(),
                                          activation ? activation->kind : WK_ACT_NONE, sens->rows(), sens->cols(), c->outputs[i]->buffer,
                                          c->outputs[i]->memory_layout.row_pitch, sens->buffer, sens->memory_layout.row_pitch, dev->buffer,
                                          dev->memory_layout.row_pitch, bias_enabled ? c->bias_gradients[i]->buffer : nullptr));
            }
            pipeline->append(1);
            // weight gradient: sens^T [O,B] * prev_output [B,I]
            blas::gemm<T>(pipeline, std::nullopt, sens, blas::Operation::transpose, prev_output, blas::Operation::no_transpose,
                          std::nullopt, c->gradients[i], nullptr);
            TensorT *next = i >= 1 ? c->sensitivities[i - 1] : input_sensitivity;
            if (!next) return;
            // sensitivity of what feeds this matrix: sens [B,O] * W [O,I]
            blas::gemm<T>(pipeline, std::nullopt, sens, blas::Operation::no_transpose, weights[i], blas::Operation::no_transpose,
                          std::nullopt, next, nullptr);
            sens = next;
        }
    }
    std::vector<TensorT *> getGradients(const void *cache) const override {
        return static_cast<const LinearCache *>(cache)->gradients;
    }
    std::vector<TensorT *> getBiasGradients(const void *cache) const override {
        if (!bias_enabled) return std::vector<TensorT *>(weights.size(), nullptr);
        return static_cast<const LinearCache *>(cache)->bias_gradients;
    }
};

// ---- Dropout -----------------------------------------------------------------------------------
// No counterpart in the reference.  random::dropout between two layers, `width` columns: every forward pass takes the layer's
// next count, which its cache keeps for the backward pass.  setTraining(false): the outputs are the inputs.
// The count is the host's, so passes captured into a graph keep the one they had then, and replays would repeat their masks.
// setStep: one element in device memory (the caller's; null: none) that the passes from then on add to their count when they run; a
// program moves it between replays by the forward passes of the layer in one, and not between a forward pass and its backward pass.
template <typename T> struct Dropout : Layer<T> {
    using TensorT = Tensor<T>;
    struct DropoutCache {
        TensorT *output = nullptr, *sensitivity = nullptr;
        uint64_t count = 0; // of the last forward pass
        double p = 0.0;     // what it dropped
        Tensor<uint64_t> *step = nullptr; // what it added to the count
    };
    const Context *context = nullptr;
    uint64_t width = 0, seed = 0;
    double p = 0.0;
    bool training = true;
    Tensor<uint64_t> *step = nullptr;
    mutable std::atomic<uint64_t> count{0};

    static Dropout *init(const Context *context, uint64_t width, double p, std::optional<uint64_t> seed = std::nullopt) {
        if (!width || !(p >= 0.0 && p <= 1.0)) throw Error(WK_E_INVALID_VALUE);
        Dropout *d = new Dropout;
        d->context = context;
        d->width = width;
        d->p = p;
        d->seed = seed ? *seed : (uint64_t)std::chrono::steady_clock::now().time_since_epoch().count();
        return d;
    }
    void setTraining(bool on) override { training = on; }
    void setStep(Tensor<uint64_t> *counter) override {
        if (counter && counter->context != context) throw Error(WK_E_UNQUAL_TENSORS_CONTEXT);
        step = counter;
    }
    void deinit(Pipeline *) override { delete this; }
    TensorT *getCachedOutput(const void *cache) const override { return static_cast<const DropoutCache *>(cache)->output; }
    std::vector<TensorT *> getWeights() const override { return {}; }
    std::vector<TensorT *> getBias() const override { return {}; }
    void *prepareCache(Pipeline *pipeline, uint64_t number_of_elements) const override {
        if (number_of_elements == 0) throw Error(WK_E_INVALID_VALUE);
        auto c = std::make_unique<DropoutCache>();
        try {
            c->output = TensorT::alloc(context, pipeline, {number_of_elements, width});
            c->sensitivity = TensorT::alloc(context, pipeline, {number_of_elements, width});
            fill::one<T>(pipeline, c->sensitivity);
        } catch (...) {
            releaseCache(pipeline, c.release());
            throw;
        }
        return c.release();
    }
    void releaseCache(Pipeline *pipeline, void *cache) const override {
        DropoutCache *c = static_cast<DropoutCache *>(cache);
        if (c->output) c->output->release(pipeline);
        if (c->sensitivity) c->sensitivity->release(pipeline);
        delete c;
    }
    TensorT *forward(Pipeline *pipeline, TensorT *input, void *cache) const override {
        DropoutCache *c = static_cast<DropoutCache *>(cache);
        helpers::eqlTensorsShape<T>(input, c->output); // a refused call takes no count
        const double drops = training ? p : 0.0;
        const uint64_t n = training ? count.fetch_add(1) : 0;
        random::dropout<T>(pipeline, input, c->output, drops, seed, n, step);
        c->p = drops; // (once the pass runs: until then the cache holds the last one's, which backward goes by)
        c->count = n;
        c->step = step;
        return c->output;
    }
    TensorT *getSensitivity(const void *cache) const override { return static_cast<const DropoutCache *>(cache)->sensitivity; }
    void backward(Pipeline *pipeline, void *cache, TensorT *, TensorT *input_sensitivity) const override {
        DropoutCache *c = static_cast<DropoutCache *>(cache);
        if (input_sensitivity) random::dropout<T>(pipeline, c->sensitivity, input_sensitivity, c->p, seed, c->count, c->step);
    }
    std::vector<TensorT *> getGradients(const void *) const override { return {}; }
    std::vector<TensorT *> getBiasGradients(const void *) const override { return {}; }
};

// ---- Sequential --------------------------------------------------------------------------------
template <typename T> struct Sequential : Layer<T> {
    using TensorT = Tensor<T>;
    struct SequentialCache {
        std::vector<void *> caches;
    };
    std::vector<Layer<T> *> layers; // owned

    // Sequential.init / append (sequential.zig:40-90): starts empty, owns what is appended
    static Sequential *init() { return new Sequential; }
    void append(Layer<T> *layer) { layers.push_back(layer); }
    void setTraining(bool on) override {
        for (Layer<T> *l : layers) l->setTraining(on);
    }
    void setStep(Tensor<uint64_t> *counter) override {
        for (Layer<T> *l : layers) l->setStep(counter);
    }
    void deinit(Pipeline *pipeline) override {
        for (Layer<T> *l : layers) l->deinit(pipeline);
        delete this;
    }
    TensorT *getCachedOutput(const void *cache) const override {
        const auto *c = static_cast<const SequentialCache *>(cache);
        return layers.back()->getCachedOutput(c->caches.back());
    }
    std::vector<TensorT *> getWeights() const override {
        std::vector<TensorT *> out;
        for (Layer<T> *l : layers)
            for (TensorT *w : l->getWeights()) out.push_back(w);
        return out;
    }
    std::vector<TensorT *> getBias() const override {
        std::vector<TensorT *> out;
        for (Layer<T> *l : layers)
            for (TensorT *b : l->getBias()) out.push_back(b);
        return out;
    }
    void *prepareCache(Pipeline *pipeline, uint64_t number_of_elements) const override {
        if (layers.empty()) throw Error(WK_E_INVALID_VALUE);
        auto c = std::make_unique<SequentialCache>();
        try {
            for (Layer<T> *l : layers) c->caches.push_back(l->prepareCache(pipeline, number_of_elements));
        } catch (...) {
            for (size_t i = 0; i < c->caches.size(); ++i) layers[i]->releaseCache(pipeline, c->caches[i]);
            throw;
        }
        return c.release();
    }
    void releaseCache(Pipeline *pipeline, void *cache) const override {
        auto *c = static_cast<SequentialCache *>(cache);
        for (size_t i = 0; i < layers.size(); ++i) layers[i]->releaseCache(pipeline, c->caches[i]);
        delete c;
    }
    // sequential.zig:214-230
    TensorT *forward(Pipeline *pipeline, TensorT *input, void *cache) const override {
        auto *c = static_cast<SequentialCache *>(cache);
        TensorT *out = input;
        for (size_t i = 0; i < layers.size(); ++i) out = layers[i]->forward(pipeline, out, c->caches[i]);
        return out;
    }
    TensorT *getSensitivity(const void *cache) const override {
        const auto *c = static_cast<const SequentialCache *>(cache);
        return layers.back()->getSensitivity(c->caches.back());
    }
    // sequential.zig:242-274: last layer to first; layer i's input is layer i-1's cached output and
    // its input gradient is layer i-1's sensitivity
    void backward(Pipeline *pipeline, void *cache, TensorT *input, TensorT *input_gradient) const override {
        auto *c = static_cast<SequentialCache *>(cache);
        for (size_t i = layers.size(); i-- > 0;) {
            TensorT *in = i == 0 ? input : layers[i - 1]->getCachedOutput(c->caches[i - 1]);
            TensorT *in_grad = i == 0 ? input_gradient : layers[i - 1]->getSensitivity(c->caches[i - 1]);
            layers[i]->backward(pipeline, c->caches[i], in, in_grad);
        }
    }
    std::vector<TensorT *> getGradients(const void *cache) const override {
        const auto *c = static_cast<const SequentialCache *>(cache);
        std::vector<TensorT *> out;
        for (size_t i = 0; i < layers.size(); ++i)
            for (TensorT *g : layers[i]->getGradients(c->caches[i])) out.push_back(g);
        return out;
    }
    std::vector<TensorT *> getBiasGradients(const void *cache) const override {
        const auto *c = static_cast<const SequentialCache *>(cache);
        std::vector<TensorT *> out;
        for (size_t i = 0; i < layers.size(); ++i)
            for (TensorT *g : layers[i]->getBiasGradients(c->caches[i])) out.push_back(g);
        return out;
    }
};

// ---- Cache (src/nn/layer/cache.zig) --------------------------------------------------------------
template <typename T> struct Cache {
    struct Slot {
        void *cache;
        const Layer<T> *layer;
    };
    std::vector<Slot> slots;
    Tensor<T> *error_tensor = nullptr;

    static Cache *init(const Context *context, Pipeline *pipeline, uint64_t number_of_elements,
                       const std::vector<const Layer<T> *> &layers) {
        if (layers.empty()) throw Error(WK_E_INVALID_VALUE);
        auto self = std::make_unique<Cache>();
        try {
            for (const Layer<T> *l : layers) self->slots.push_back({l->prepareCache(pipeline, number_of_elements), l});
            const Slot &last = self->slots.back();
            self->error_tensor = Tensor<T>::alloc(context, pipeline, last.layer->getSensitivity(last.cache)->dimensions.shape);
        } catch (...) {
            for (const Slot &s : self->slots) s.layer->releaseCache(pipeline, s.cache);
            throw;
        }
        return self.release();
    }
    void *getLayerCache(size_t index) const { return slots[index].cache; }
    void deinit(Pipeline *pipeline) {
        for (const Slot &s : slots) s.layer->releaseCache(pipeline, s.cache);
        error_tensor->release(pipeline);
        delete this;
    }
};

// ---- log probabilities of tokens (no counterpart in the reference) --------------------------------------
// Results and workspace of wk_token_logprobs for {rows, vocab} logits: for scoring and serving (with the `top` likeliest
// tokens) and for training.  T: f32, f64, F16, BF16; results are f32 (f64 for f64).  Both are overwritten by the next forward
// pass: passes on one object are for one pipeline, or ordered.
template <typename T> struct TokenLogProbs {
    using S = std::conditional_t<std::is_same_v<T, double>, double, float>;
    uint64_t rows = 0, vocab = 0;
    uint32_t top = 0;
    Tensor<S> *logprob = nullptr, *lse = nullptr, *entropy = nullptr; // {rows}
    Tensor<int32_t> *top_ids = nullptr;                               // {rows * top}, row by row; null without alternatives
    Tensor<S> *top_logprobs = nullptr;
    Tensor<S> *minus_one = nullptr; // {rows}: the gradient of a loss that is the sum of -logprob
    wk_device *device = nullptr;
    void *workspace = nullptr;
    size_t workspace_bytes = 0;

    static TokenLogProbs *init(const Context *context, Pipeline *pipeline, uint64_t rows, uint64_t vocab, uint32_t top = 0) {
        if (!rows || !vocab || top > WK_TOKEN_TOP_MAX || top > vocab) throw Error(WK_E_INVALID_VALUE);
        TokenLogProbs *t = new TokenLogProbs;
        t->rows = rows;
        t->vocab = vocab;
        t->top = top;
        t->device = context->device;
        try {
            for (Tensor<S> **r : {&t->logprob, &t->lse, &t->entropy, &t->minus_one}) *r = Tensor<S>::alloc(context, pipeline, {rows});
            fill::constant<S>(pipeline, t->minus_one, S(-1));
            if (top) {
                t->top_ids = Tensor<int32_t>::alloc(context, pipeline, {rows * top});
                t->top_logprobs = Tensor<S>::alloc(context, pipeline, {rows * top});
            }
            t->workspace_bytes = wk_token_logprobs_workspace_bytes(core::getTypeIndex<T>(), rows, vocab, top);
            if (t->workspace_bytes) check(wk_malloc(t->device, t->workspace_bytes, &t->workspace));
        } catch (...) {
            t->deinit(pipeline);
            throw;
        }
        return t;
    }
    void deinit(Pipeline *pipeline) {
        pipeline->waitAndCleanup();
        for (Tensor<S> *r : {logprob, lse, entropy, minus_one, top_logprobs})
            if (r) r->release(pipeline);
        if (top_ids) top_ids->release(pipeline);
        if (workspace) wk_free(device, workspace);
        delete this;
    }
    template <typename Id> void validate(const Tensor<T> *logits, const Tensor<Id> *targets) const {
        static_assert(std::is_same_v<Id, int32_t> || std::is_same_v<Id, int64_t>);
        if (logits->context != lse->context || (targets && targets->context != lse->context)) throw Error(WK_E_UNQUAL_TENSORS_CONTEXT);
        if (logits->depth() != 1 || logits->rows() != rows || logits->cols() != vocab) throw Error(WK_E_UNQUAL_TENSORS_SHAPE);
        if (targets && targets->dimensions.shape != std::vector<uint64_t>{rows}) throw Error(WK_E_UNQUAL_TENSORS_SHAPE);
    }
    // targets null: no logprob
    template <typename Id> void forward(Pipeline *pipeline, const Tensor<T> *logits, const Tensor<Id> *targets) {
        validate(logits, targets);
        check(wk_token_logprobs(pipeline->command_queue->stream, core::getTypeIndex<T>(), rows, vocab, logits->buffer,
                                logits->memory_layout.row_pitch, targets ? targets->buffer : nullptr, core::getTypeIndex<Id>(),
                                targets ? logprob->buffer : nullptr, lse->buffer, entropy->buffer, top,
                                top ? static_cast<int32_t *>(top_ids->buffer) : nullptr, top ? top_logprobs->buffer : nullptr, workspace,
                                workspace_bytes));
        pipeline->append(1);
    }
    // after forward on the same logits; logits_grad may be logits; logprob_grad, entropy_grad {rows}, either null
    template <typename Id>
    void backward(Pipeline *pipeline, const Tensor<T> *logits, const Tensor<Id> *targets, const Tensor<S> *logprob_grad,
                  const Tensor<S> *entropy_grad, Tensor<T> *logits_grad) {
        validate(logits, targets);
        helpers::eqlTensorsShape<T>(logits, logits_grad);
        for (const Tensor<S> *g : {logprob_grad, entropy_grad})
            if (g && g->dimensions.shape != std::vector<uint64_t>{rows}) throw Error(WK_E_UNQUAL_TENSORS_SHAPE);
        check(wk_token_logprobs_grad(pipeline->command_queue->stream, core::getTypeIndex<T>(), rows, vocab, logits->buffer,
                                     logits->memory_layout.row_pitch, targets ? targets->buffer : nullptr, core::getTypeIndex<Id>(), lse->buffer,
                                     entropy->buffer, logprob_grad ? logprob_grad->buffer : nullptr,
                                     entropy_grad ? entropy_grad->buffer : nullptr, logits_grad->buffer, logits_grad->memory_layout.row_pitch));
        pipeline->append(1);
    }
};

// ---- loss ------------------------------------------------------------------------------------------
namespace loss {
// No counterpart in the reference: the loss of a network whose outputs are logits over a vocabulary, minus the log probability
// of each row's target.  As mse does, the derivative goes into the last layer's sensitivity without a factor 1 / rows; error_result,
// when wanted, is the mean over all rows (this synchronises the pipeline).  A negative target counts nothing and has no gradient.
template <typename T, typename Id>
void tokens(bool calculate_derivative, Pipeline *pipeline, Tensor<T> *output, Tensor<Id> *targets, TokenLogProbs<T> *state,
            const Cache<T> *cache, T *error_result) {
    if (!targets) throw Error(WK_E_INVALID_VALUE);
    const auto &last = cache->slots.back();
    Tensor<T> *sens = last.layer->getSensitivity(last.cache);
    helpers::eqlTensorsShape<T>(output, sens);
    state->forward(pipeline, output, targets);
    if (calculate_derivative)
        state->template backward<Id>(pipeline, output, targets, state->minus_one, nullptr, sens);
    if (error_result) *error_result = -math::mean<T>(pipeline, state->logprob);
}

// mse (src/nn/loss/mse.zig:63-132): error_tensor = (expected - output)^2; with calculate_derivative
// the last layer's sensitivity receives -2 (expected - output); error_result, when wanted, is the
// mean of error_tensor (this synchronises the pipeline, as math.mean does).
template <typename T>
void mse(bool calculate_derivative, Pipeline *pipeline, Tensor<T> *output, Tensor<T> *expected, const Cache<T> *cache,
         T *error_result) {
    Tensor<T> *err = cache->error_tensor;
    helpers::eqlTensorsShape<T>(output, expected);
    helpers::eqlTensorsShape<T>(err, output);
    Tensor<T> *sens = nullptr;
    if (calculate_derivative) {
        const auto &last = cache->slots.back();
        sens = last.layer->getSensitivity(last.cache);
    }
    const uint64_t shape3[3] = {output->depth(), output->rows(), output->cols()};
    check(wk_mse(pipeline->command_queue->stream, core::getTypeIndex<T>(), shape3, output->buffer, output->memory_layout.row_pitch,
                 output->memory_layout.slice_pitch, expected->buffer, expected->memory_layout.row_pitch,
                 expected->memory_layout.slice_pitch, err->buffer, err->memory_layout.row_pitch, err->memory_layout.slice_pitch,
                 sens ? sens->buffer : nullptr, sens ? sens->memory_layout.row_pitch : 0, sens ? sens->memory_layout.slice_pitch : 0));
    pipeline->append(1);
    if (error_result) *error_result = math::mean<T>(pipeline, err);
}
} // namespace loss

// ---- optimizers ----------------------------------------------------------------------------------
namespace optimizers {
template <typename T> struct Optimizer {
    virtual ~Optimizer() = default;
    virtual void step(Pipeline *pipeline, const Cache<T> *cache) = 0;
    virtual void zero(Pipeline *pipeline) = 0;
    virtual void deinit(Pipeline *pipeline) = 0;
};

// GD (src/nn/optimizers/gd.zig): w += (-lr) * g with blas.axpy, weights then biases, slot by slot
template <typename T> struct GD : Optimizer<T> {
    T lr; // stored negated, as gd.zig:39 does
    static GD *init(T lr) {
        GD *o = new GD;
        o->lr = -lr;
        return o;
    }
    void step(Pipeline *pipeline, const Cache<T> *cache) override {
        for (const auto &slot : cache->slots) {
            auto w = slot.layer->getWeights();
            auto g = slot.layer->getGradients(slot.cache);
            for (size_t i = 0; i < w.size(); ++i) blas::axpy<T>(pipeline, g[i], lr, w[i]);
            auto b = slot.layer->getBias();
            auto bg = slot.layer->getBiasGradients(slot.cache);
            for (size_t i = 0; i < b.size(); ++i)
                if (b[i] && bg[i]) blas::axpy<T>(pipeline, bg[i], lr, b[i]);
        }
    }
    void zero(Pipeline *) override {}
    void deinit(Pipeline *) override { delete this; }
};

// Adam: first/second moment tensors are created lazily with the shape of each parameter.
template <typename T> struct Adam : Optimizer<T> {
    double lr = 1e-3, beta1 = 0.9, beta2 = 0.999, eps = 0.0;
    uint64_t t = 0;
    std::vector<std::pair<Tensor<T> *, Tensor<T> *>> state; // (m, v) per parameter, in visiting order

    static Adam *init(double lr, double beta1 = 0.9, double beta2 = 0.999, double eps = -1.0) {
        Adam *o = new Adam;
        o->lr = lr;
        o->beta1 = beta1;
        o->beta2 = beta2;
        o->eps = eps >= 0.0 ? eps : (double)std::numeric_limits<T>::epsilon(); // the siblings' +FLT_EPSILON (rmsprop.cl:54)
        return o;
    }
    // one parameter tensor's entry of the step's update list (its moments are created on first sight)
    void collect(Pipeline *pipeline, size_t &index, Tensor<T> *w, Tensor<T> *g, std::vector<wk_adam_tensor> &list) {
        if (index == state.size()) {
            Tensor<T> *m = Tensor<T>::alloc(w->context, pipeline, w->dimensions.shape);
            Tensor<T> *v = nullptr;
            try {
                v = Tensor<T>::alloc(w->context, pipeline, w->dimensions.shape);
            } catch (...) {
                m->release(pipeline);
                throw;
            }
            state.push_back({m, v});
        }
        Tensor<T> *m = state[index].first, *v = state[index].second;
        helpers::eqlTensorsShape<T>(w, g);
        helpers::eqlTensorsShape<T>(w, m);
        wk_adam_tensor t{};
        t.w = w->buffer; t.g = g->buffer; t.m = m->buffer; t.v = v->buffer;
        t.shape3[0] = w->depth(); t.shape3[1] = w->rows(); t.shape3[2] = w->cols();
        t.w_row_pitch = w->memory_layout.row_pitch; t.w_slice_pitch = w->memory_layout.slice_pitch;
        t.g_row_pitch = g->memory_layout.row_pitch; t.g_slice_pitch = g->memory_layout.slice_pitch;
        t.mv_row_pitch = m->memory_layout.row_pitch; t.mv_slice_pitch = m->memory_layout.slice_pitch;
        list.push_back(t);
        ++index;
    }
    void step(Pipeline *pipeline, const Cache<T> *cache) override {
        ++t;
        size_t index = 0;
        std::vector<wk_adam_tensor> list;
        for (const auto &slot : cache->slots) {
            auto w = slot.layer->getWeights();
            auto g = slot.layer->getGradients(slot.cache);
            for (size_t i = 0; i < w.size(); ++i) collect(pipeline, index, w[i], g[i], list);
            auto b = slot.layer->getBias();
            auto bg = slot.layer->getBiasGradients(slot.cache);
            for (size_t i = 0; i < b.size(); ++i)
                if (b[i] && bg[i]) collect(pipeline, index, b[i], bg[i], list);
        }
        check(wk_adam_step_multi(pipeline->command_queue->stream, core::getTypeIndex<T>(), (uint32_t)list.size(), list.data(), lr, beta1,
                                 beta2, eps, t));
        pipeline->append(1);
    }
    void zero(Pipeline *pipeline) override {
        for (auto &mv : state) {
            fill::zeroes<T>(pipeline, mv.first);
            fill::zeroes<T>(pipeline, mv.second);
        }
        t = 0;
    }
    void deinit(Pipeline *pipeline) override {
        for (auto &mv : state) {
            mv.first->release(pipeline);
            mv.second->release(pipeline);
        }
        delete this;
    }
};
} // namespace optimizers

} // namespace nn
} // namespace wekua
