"""JSON weight import of a layer whose routing has a bias for balance (host logic, CPU only)."""
import numpy as np
import pytest

from tests.test_weights_json import FakeLayer, W, _arrays

D, H, E = 6, 4, 3
B = np.float32([0.25, -0.5, 0.125])


class Balanced(FakeLayer):
    hasBalance = True
    balance = None

    def set_balance(self, b):
        self.balance = b


@pytest.mark.parametrize("scheme", ["omega", "deepseek"])
def test_round_trip(scheme):
    a = dict(_arrays(D, H, E, 0, False), balance=B)
    m = W.export_moe_weights(a, layer_index=2, scheme=scheme)
    lay = Balanced(D, H, E, 0)
    assert W.load_moe_weights(lay, m, layer_index=2, scheme=scheme) == ["layers.2.ffn_norm.weight" if scheme == "omega" else "model.layers.2.post_attention_layernorm.weight"]
    assert np.array_equal(lay.balance, B) and lay.balance.dtype == np.float32 and lay.bias is None and np.array_equal(lay.gate, a["Wg"])
    plain = FakeLayer(D, H, E, 0)                      # a layer without one leaves it
    W.load_moe_weights(plain, m, layer_index=2, scheme=scheme)
    assert plain.bias is None
    del m[[k for k in m if "balance" in k or "correction" in k][0]]
    with pytest.raises(RuntimeError, match="is null"):
        W.load_moe_weights(Balanced(D, H, E, 0), m, layer_index=2, scheme=scheme)
    assert Balanced(D, H, E, 0).balance is None


def test_the_gates_bias_beside_it():
    a = dict(_arrays(D, H, E, 0, True), balance=B)
    lay = Balanced(D, H, E, 0, True)
    W.load_moe_weights(lay, W.export_moe_weights(a, scheme="omega"), scheme="omega")
    assert np.array_equal(lay.balance, B) and np.array_equal(lay.bias, a["bg"])
    with pytest.raises(ValueError, match="one name"):
        W.export_moe_weights(a, scheme="deepseek")
    # one name: the routing's, which the choice alone reads
    m = W.export_moe_weights(dict(a, balance=None), scheme="deepseek")
    lay = Balanced(D, H, E, 0, True)
    W.load_moe_weights(lay, m, scheme="deepseek")
    assert np.array_equal(lay.balance, a["bg"]) and lay.bias is None


def test_a_scheme_without_a_name():
    a = dict(_arrays(D, H, E, 0, False), balance=B)
    m = W.export_moe_weights(a, scheme="mixtral")
    lay = Balanced(D, H, E, 0)
    W.load_moe_weights(lay, m, scheme="mixtral")
    assert lay.balance is None
