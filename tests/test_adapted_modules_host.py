"""Adapters and the other swaps in modules that hold their layers in unusual ways.  No GPU needed: without selected rows an adapted linear is its linear, and the layers' forward passes are stood in for."""
import copy

import pytest
import torch
import torch.nn as nn

import float8_experimental_amd as f8

x = torch.randn(2, 5, 16, generator=torch.Generator().manual_seed(0))
ATTENTION = lambda: nn.MultiheadAttention(16, 2, batch_first=True)
LAYER = lambda: nn.TransformerEncoderLayer(16, 2, 32, batch_first=True)
OF_TORCH = {  # module, its arguments, the linears that it always calls
    "attention": (ATTENTION, (x, x, x), []),
    "encoder layer": (LAYER, (x,), []),
    "encoder": (lambda: nn.TransformerEncoder(LAYER(), 2), (x,), []),
    "decoder layer": (lambda: nn.TransformerDecoderLayer(16, 2, 32, batch_first=True), (x, x), ["linear1", "linear2"]),
    "both": (lambda: nn.Sequential(LAYER(), nn.Linear(16, 4)), (x,), ["1"]),
    "adaptive softmax": (lambda: nn.AdaptiveLogSoftmaxWithLoss(16, 30, [5, 10]), (torch.randn(4, 16), torch.tensor([1, 7, 20, 29])), ["head", "tail.0.0", "tail.0.1", "tail.1.0", "tail.1.1"]),
}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("training", [False, True])
@pytest.mark.parametrize("name", list(OF_TORCH))
def test_modules_that_read_the_weights_of_their_linears(monkeypatch, name, training, grad):
    make, args, called = OF_TORCH[name]
    torch.manual_seed(0)
    plain = make().train(training).requires_grad_(False)  # (as adapting it freezes it: torch chooses its path by that)
    adapted = f8.adapt_linears(copy.deepcopy(plain), 3, 2)
    names = {id(m): fqn for fqn, m in adapted.named_modules() if isinstance(m, f8.AdaptedLinear)}
    assert list(names.values()) == called
    seen, forward = [], f8.AdaptedLinear.forward
    monkeypatch.setattr(f8.AdaptedLinear, "forward", lambda self, input: seen.append(names[id(self)]) or forward(self, input))
    first = lambda out: out[0] if isinstance(out, tuple) else out
    with torch.set_grad_enabled(grad):
        torch.manual_seed(1)
        want = first(plain(*args))
        torch.manual_seed(1)
        got = first(adapted(*args))
    assert torch.equal(got, want) and sorted(seen) == sorted(called)  # none of the adapters is passed by


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("make, fqn", [(ATTENTION, "out_proj"), (LAYER, "linear1"), (LAYER, "linear2"), (LAYER, "self_attn.out_proj"), (lambda: nn.Transformer(16, 2, 1, 1, 32), "encoder.layers.0.linear1")])
def test_a_filter_that_asks_for_what_is_not_called(make, fqn):
    model = nn.Sequential(nn.Linear(4, 4), make())
    for ask in (lambda m, name: True, lambda m, name: name == f"1.{fqn}"):
        with pytest.raises(ValueError, match="reads the weight"):
            f8.adapt_linears(model, 3, 2, module_filter_fn=ask)
        assert type(model[0]) is nn.Linear and all(p.requires_grad for p in model.parameters())  # nothing has been changed
    f8.adapt_linears(model, 3, 2, module_filter_fn=lambda m, name: name == "0")
    assert type(model[0]) is f8.AdaptedLinear and sum(isinstance(m, f8.AdaptedLinear) for m in model.modules()) == 1


class Held(nn.Module):
    """One layer of each kind under two names and by two modules, one of them held twice itself."""

    def __init__(self, layer):
        super().__init__()
        self.a, self.absent, self.inner = layer, None, nn.Sequential(layer, nn.Sequential(layer))
        self.b, self.again = layer, self.inner

    def forward(self, x):
        return self.b(self.again(self.inner(self.a(x))))

    def layers(self):
        return [self.a, self.b, self.inner[0], self.inner[1][0], self.again[0]]


def test_a_linear_under_several_names_has_one_set_of_adapters():
    linear = nn.Linear(16, 16)
    model = f8.adapt_linears(Held(linear), 3, 2)
    first, *others = model.layers()
    assert type(first) is f8.AdaptedLinear and first.linear is linear and all(m is first for m in others)
    assert len([p for p in model.parameters() if p.requires_grad]) == 2 and model(x).shape == x.shape
    again = f8.adapt_linears(model, 3, 4)
    assert again is model and all(m is first for m in model.layers()) and first.linear is linear
    two = nn.Sequential(nn.Linear(4, 4), nn.Linear(4, 4))
    two[1].weight = two[0].weight  # a shared weight is not a shared linear
    f8.adapt_linears(two, 3, 2)
    assert two[0] is not two[1] and two[0].linear.weight is two[1].linear.weight and two[0].adapter_a is not two[1].adapter_a


def test_names_that_the_filter_leaves_out_stay_as_they_are():
    linear = nn.Linear(16, 16)
    model = f8.adapt_linears(Held(linear), 3, 2, module_filter_fn=lambda m, fqn: fqn in ("b", "inner.1.0"))
    assert model.a is linear and model.inner[0] is linear and type(model.b) is f8.AdaptedLinear and model.inner[1][0] is model.b


@pytest.mark.parametrize("convert, plain, own", [(f8.convert_rms_norms, lambda: nn.RMSNorm(16), f8.RMSNorm), (f8.convert_layer_norms, lambda: nn.LayerNorm(16), f8.LayerNorm),
                                                 (f8.convert_dropouts, lambda: nn.Dropout(0.25), f8.Dropout)])
def test_a_layer_under_several_names_is_converted_under_all_of_them(convert, plain, own):
    model = Held(plain())
    params = list(model.parameters())
    assert convert(model) is model
    first, *others = model.layers()
    assert type(first) is own and all(m is first for m in others) and model.absent is None
    assert all(p is q for p, q in zip(model.parameters(), params)) and convert(model) is model and model.a is first
    assert type(convert(plain())) is own

    class Of(type(plain())):
        pass

    of = nn.Sequential(Of(0.5) if own is f8.Dropout else Of(16))
    assert type(convert(of)[0]) is Of  # a subclass may do something else


def test_dropout_in_place_is_refused():
    for make in (lambda: f8.Dropout(0.5, inplace=True), lambda: f8.Dropout(0.5, True), lambda: f8.Dropout.from_float(nn.Dropout(0.5, True)), lambda: f8.convert_dropouts(nn.Sequential(nn.Dropout(0.5, True)))):
        with pytest.raises(NotImplementedError, match="in place"):
            make()
    layer = f8.Dropout(0.25, inplace=False)
    assert layer.p == 0.25 and not layer.inplace and f8.Dropout().p == 0.5 and f8.Dropout(p=0.1).p == 0.1
    with pytest.raises(ValueError):
        f8.Dropout(1.5)
