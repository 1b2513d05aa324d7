// extern "C" boundary of the sequence operators (include/b200fft.h).
#include <cmath>
#include <cstring>

#include "../capi_guard.hpp"
#include "sequence.hpp"

using namespace b200fft;

struct b200fft_layer_norm {
    LayerNorm n;
};
struct b200fft_linear_attention {
    LinearAttention a;
};

extern "C" {

b200fft_status b200fft_layer_norm_config_init(b200fft_layer_norm_config *config, uint64_t rows, uint64_t features) {
    return guarded([&] {
        need(config, "config");
        std::memset(config, 0, sizeof(*config));
        config->rows = rows;
        config->features = features;
        config->epsilon = 1e-5f;
    });
}

b200fft_status b200fft_layer_norm_config_validate(const b200fft_layer_norm_config *config) {
    return guarded([&] {
        need(config, "config");
        LayerNorm::from_c(*config);
    });
}

b200fft_status b200fft_layer_norm_build(const b200fft_layer_norm_config *config, const b200fft_device_profile *device,
                                        b200fft_layer_norm **layer_norm) {
    return guarded([&] {
        need(config, "config");
        need(device, "device");
        need(layer_norm, "layer_norm");
        *layer_norm = nullptr;
        *layer_norm = new b200fft_layer_norm{LayerNorm::from_c(*config)};
    });
}

void b200fft_layer_norm_destroy(b200fft_layer_norm *layer_norm) { delete layer_norm; }

uint64_t b200fft_layer_norm_backward_workspace_bytes(const b200fft_layer_norm *layer_norm) {
    return layer_norm ? layer_norm->n.backward_workspace() : 0;
}

b200fft_status b200fft_execute_layer_norm(b200fft_context *context, b200fft_layer_norm *layer_norm, const void *input,
                                          const void *weight, const void *bias, void *output, float *mean, float *rstd,
                                          void *stream) {
    return guarded([&] {
        need(context, "context");
        need(layer_norm, "layer_norm");
        NormParams p{};
        p.x = input;
        p.w = weight;
        p.b = bias;
        p.y = output;
        p.mean = mean;
        p.rstd = rstd;
        execute_layer_norm(context->ctx, layer_norm->n, p, static_cast<cudaStream_t>(stream));
    });
}

b200fft_status b200fft_execute_layer_norm_backward(b200fft_context *context, b200fft_layer_norm *layer_norm,
                                                   const void *input, const void *weight, const float *mean,
                                                   const float *rstd, const void *output_gradient,
                                                   void *input_gradient, void *weight_gradient, void *bias_gradient,
                                                   void *workspace, void *stream) {
    return guarded([&] {
        need(context, "context");
        need(layer_norm, "layer_norm");
        NormGradParams p{};
        p.x = input;
        p.w = weight;
        p.mean = mean;
        p.rstd = rstd;
        p.dy = output_gradient;
        p.dx = input_gradient;
        p.dw = weight_gradient;
        p.db = bias_gradient;
        execute_layer_norm_grad(context->ctx, layer_norm->n, p, workspace, static_cast<cudaStream_t>(stream));
    });
}

b200fft_status b200fft_linear_attention_config_init(b200fft_linear_attention_config *config, uint64_t length,
                                                    uint64_t heads, uint64_t key_dim, uint64_t value_dim) {
    return guarded([&] {
        need(config, "config");
        std::memset(config, 0, sizeof(*config));
        config->batch_count = 1;
        config->length = length;
        config->heads = heads;
        config->key_value_heads = heads;
        config->key_dim = key_dim;
        config->value_dim = value_dim;
        config->scale = key_dim ? 1.f / std::sqrt((float)key_dim) : 1.f;
    });
}

b200fft_status b200fft_linear_attention_config_validate(const b200fft_linear_attention_config *config) {
    return guarded([&] {
        need(config, "config");
        LinearAttention::from_c(*config);
    });
}

b200fft_status b200fft_linear_attention_build(const b200fft_linear_attention_config *config,
                                              const b200fft_device_profile *device,
                                              b200fft_linear_attention **attention) {
    return guarded([&] {
        need(config, "config");
        need(device, "device");
        need(attention, "attention");
        *attention = nullptr;
        *attention = new b200fft_linear_attention{LinearAttention::from_c(*config)};
    });
}

void b200fft_linear_attention_destroy(b200fft_linear_attention *attention) { delete attention; }

uint64_t b200fft_linear_attention_workspace_bytes(const b200fft_linear_attention *attention) {
    return attention ? attention->a.workspace() : 0;
}

uint64_t b200fft_linear_attention_backward_workspace_bytes(const b200fft_linear_attention *attention) {
    return attention ? attention->a.backward_workspace() : 0;
}

b200fft_status b200fft_execute_linear_attention(b200fft_context *context, b200fft_linear_attention *attention,
                                                const b200fft_linear_attention_buffers *buffers, void *workspace,
                                                void *stream) {
    return guarded([&] {
        need(context, "context");
        need(attention, "attention");
        need(buffers, "buffers");
        execute_linear_attention(context->ctx, attention->a, *buffers, workspace, static_cast<cudaStream_t>(stream));
    });
}

b200fft_status b200fft_execute_linear_attention_backward(b200fft_context *context, b200fft_linear_attention *attention,
                                                         const b200fft_linear_attention_gradients *gradients,
                                                         void *workspace, void *stream) {
    return guarded([&] {
        need(context, "context");
        need(attention, "attention");
        need(gradients, "gradients");
        execute_linear_attention_grad(context->ctx, attention->a, *gradients, workspace,
                                      static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
