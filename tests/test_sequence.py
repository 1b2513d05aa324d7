"""Configurations of the sequence operators: refusals and sizes, without a GPU."""
import pytest


def refuses(V, variant, call):
    with pytest.raises(V.VkFftError) as e:
        call()
    assert e.value.variant == variant


def test_layer_norm_config(V, cuda_profile):
    V.LayerNormConfig(3, 5).validate()
    refuses(V, "ZeroBatchCount", V.LayerNormConfig(0, 4).validate)
    refuses(V, "ZeroLength", V.LayerNormConfig(4, 0).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(4, 8).with_input_row_stride(7).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(4, 8).with_output_row_stride(7).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(4, 8).with_epsilon(-1.0).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(4, 8).with_epsilon(float("nan")).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(4, 8).with_element_type(3).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(4, 8).with_parameter_type(-1).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(4, 1 << 40).validate)
    refuses(V, "ValueOutOfRange", V.LayerNormConfig(1 << 39, 1 << 20).validate)
    refuses(V, "ValueOutOfRange", lambda: V.LayerNormIr.build(V.LayerNormConfig(4, 8).with_epsilon(-1.0), cuda_profile))
    ir = V.LayerNormIr.build(V.LayerNormConfig(100, 64), cuda_profile)
    assert ir.workspace_bytes == 0 and ir.backward_workspace_bytes >= 2 * 64 * 4


def test_linear_attention_config(V, cuda_profile):
    make = lambda *a: V.LinearAttentionConfig(*a)  # noqa: E731
    make(5, 4, 16, 32).with_key_value_heads(2).validate()
    for sizes in ((0, 4, 16, 16), (5, 0, 16, 16), (5, 4, 0, 16), (5, 4, 16, 0)):
        refuses(V, "ZeroLength", make(*sizes).validate)
    refuses(V, "ZeroLength", make(5, 4, 16, 16).with_key_value_heads(0).validate)
    refuses(V, "ZeroBatchCount", make(5, 4, 16, 16).with_batch_count(0).validate)
    refuses(V, "ValueOutOfRange", make(5, 4, 16, 16).with_key_value_heads(3).validate)
    refuses(V, "ValueOutOfRange", make(5, 4, 16, 16).with_key_value_heads(8).validate)
    refuses(V, "UnsupportedKernelPath", make(5, 4, 257, 16).validate)
    refuses(V, "UnsupportedKernelPath", make(5, 4, 16, 257).validate)
    refuses(V, "ValueOutOfRange", make(5, 4, 16, 16).with_element_type(7).validate)
    refuses(V, "ValueOutOfRange", make(5, 4, 16, 16).with_scale(float("inf")).validate)
    refuses(V, "ValueOutOfRange", make(1 << 31, 4, 16, 16).validate)
    refuses(V, "ValueOutOfRange", make(5, 4, 16, 16).with_query_strides(0, 15, 16).validate)
    refuses(V, "ValueOutOfRange", make(5, 4, 16, 16).with_output_strides(0, 64, 8).validate)
    refuses(V, "ValueOutOfRange", make(5, 4, 16, 16).with_key_strides(0, 1 << 50, 16).validate)
    refuses(V, "ArithmeticOverflow", make(1 << 30, 4, 16, 16).with_key_strides(0, 1 << 46, 16).validate)
    with_default = make(5, 4, 16, 16)
    assert abs(with_default._s.scale - 0.25) < 1e-7
    ir = V.LinearAttentionIr.build(make(5, 4, 16, 32).with_key_value_heads(2), cuda_profile)
    assert ir.workspace_bytes >= 0 and ir.backward_workspace_bytes >= 5 * 4 * (16 + 32) * 4


def test_configurations_are_values(V):
    a = V.LinearAttentionConfig(5, 4, 16, 16)
    b = a.with_batch_count(3).with_query_strides(1, 64, 16)
    assert a._s.batch_count == 1 and b._s.batch_count == 3 and list(a._s.query_strides) == [0, 0, 0]
