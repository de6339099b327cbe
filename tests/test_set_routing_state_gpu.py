"""mgpt_moe_set_routing between two calls that belong together: what was computed under the other setting is refused, or stays what it was."""
import pytest
import torch

from mgpt_b200 import MoELayer, MoeError, _lib

pytestmark = pytest.mark.gpu


def _layer(C=64, H=64, E=8, k=2, mode="bf16", seed=0):
    g = torch.Generator().manual_seed(seed)
    layer = MoELayer(C, H, E, k, mode=mode)
    layer.load_parameters([(torch.randn(p.shape, generator=g) * (p.shape[0] ** -0.5 if p.shape[0] > 1 else 0.1)).numpy() for p in layer.get_parameters()])
    return layer


def _x(n, C, seed=1):
    return torch.randn(n, C, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).bfloat16()


@pytest.mark.parametrize("first,then", [((), ("sigmoid",)), (("sigmoid",), ()), (("sigmoid",), ("softmax",))])
def test_stage_calls_do_not_mix_settings(first, then):
    layer, x = _layer(), _x(100, 64)
    lib, h, stream = layer.lib, layer._h, layer._stream()
    ws = torch.empty(int(lib.mgpt_moe_stage_workspace_bytes(h, 100, 1)), dtype=torch.uint8, device="cuda")
    rows = torch.zeros(100 * 2 + 8 * 128, 64, dtype=torch.bfloat16, device="cuda")

    def plan():
        _lib.check(lib.mgpt_moe_route_plan(h, x.data_ptr(), 100, _lib.IO_BF16, ws.data_ptr(), ws.numel(), stream))

    def call(f, *args):
        _lib.check(f(h, *args, ws.data_ptr(), ws.numel(), stream))

    layer.set_routing(*first)
    plan()
    layer.set_routing(*then)
    with pytest.raises(MoeError, match="set after route_plan"):
        _lib.check(lib.mgpt_moe_route_rows(h, x.data_ptr(), _lib.IO_BF16, ws.data_ptr(), ws.numel(), rows.data_ptr(), stream))
    with pytest.raises(MoeError):
        call(lib.mgpt_moe_route_backward, x.data_ptr(), rows.data_ptr(), torch.empty_like(x).data_ptr(), _lib.IO_BF16)
    plan()
    _lib.check(lib.mgpt_moe_route_rows(h, x.data_ptr(), _lib.IO_BF16, ws.data_ptr(), ws.numel(), rows.data_ptr(), stream))
    y = torch.empty_like(x)
    call(lib.mgpt_moe_combine, rows.data_ptr(), y.data_ptr(), _lib.IO_BF16)
    layer.set_routing(*first)
    with pytest.raises(MoeError):
        call(lib.mgpt_moe_combine_backward, rows.data_ptr(), x.data_ptr(), _lib.IO_BF16, rows.data_ptr())


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_views_are_of_the_forward_that_filled_them(mode):
    layer, x = _layer(mode=mode), _x(100, 64)
    x = x.float() if mode == "fp32" else x

    def views():
        return [layer.workspace_view(name, torch.float32, (100, 8)).clone() for name in ("logits", "probs")]

    layer.forward(x)
    logits, probs = views()
    want = x.double() @ layer.get_parameters()[0].double() + layer.get_parameters()[1].double()
    assert (logits - want).abs().max() < 1e-4 and (probs - torch.softmax(want, 1)).abs().max() < 1e-4
    layer.set_routing("sigmoid")
    assert torch.equal(views()[0], logits) and torch.equal(views()[1], probs)
    layer.forward(x)                                                    # the router's product and its own softmax are the same
    assert torch.equal(views()[0], logits) and torch.equal(views()[1], probs)
    saved = layer.save_routing()
    layer._ws.zero_()
    layer.recompute_into(x, torch.empty_like(x), saved)                 # brings the logits back, which backward reads
    assert torch.equal(views()[0], logits)
    layer.set_routing()
    assert torch.equal(views()[0], logits)


def test_saved_routing_in_memory_of_any_alignment():
    layer, x = _layer(), _x(100, 64)
    lib, h, stream = layer.lib, layer._h, layer._stream()
    size = int(lib.mgpt_moe_routing_bytes(h, 100))
    for how in ((), ("sigmoid",)):
        layer.set_routing(*how)
        y = layer.forward(x).clone()
        dx = layer.backward(x).clone()
        for at in (0, 4, 1):
            buffer = torch.zeros(size + 16, dtype=torch.uint8, device="cuda")
            layer.forward(x)
            _lib.check(lib.mgpt_moe_save_routing(h, buffer.data_ptr() + at, stream))
            layer._ws.zero_()
            again = torch.empty_like(x)
            _lib.check(lib.mgpt_moe_forward_with_routing(h, x.data_ptr(), again.data_ptr(), 100, _lib.IO_BF16, layer._ws.data_ptr(), layer._ws.numel(),
                                                         buffer.data_ptr() + at, stream))
            assert torch.equal(again, y) and torch.equal(layer.backward(x), dx)
            layer.check_status()


def test_counts_of_the_last_forward_stay_readable():
    layer, x = _layer(), _x(100, 64)
    layer.set_routing("sigmoid")
    with pytest.raises(MoeError):                                       # there has been none
        layer.get_expert_counts()
    layer.forward(x)
    counts = layer.get_expert_counts()
    assert sum(counts) == 200
    for how in (("softmax",), (), ("sigmoid",)):
        layer.set_routing(*how)
        assert layer.get_expert_counts() == counts
    layer.forward_inference(x[:50].contiguous())
    counts = layer.get_expert_counts()
    layer.set_routing()
    assert sum(counts) == 100 and layer.get_expert_counts() == counts


@pytest.mark.parametrize("at", [0, 4])
def test_a_saved_routing_of_another_setting_is_reported(at):
    layer, x = _layer(), _x(100, 64)
    lib, h, stream = layer.lib, layer._h, layer._stream()
    size = int(lib.mgpt_moe_routing_bytes(h, 100))
    bias = torch.zeros(8, device="cuda")
    settings = [{}, dict(score="sigmoid"), dict(score="softmax"), dict(score="sigmoid", renormalise=True), dict(score="sigmoid", scale=2.0), dict(score="sigmoid", bias=bias),
                dict(score="sigmoid", groups=4, top_groups=2), dict(score="sigmoid", groups=4, top_groups=2, group_top=1)]
    saved = []
    for how in settings:
        layer.set_routing(**how)
        layer.forward(x)
        saved.append(torch.zeros(size + 16, dtype=torch.uint8, device="cuda"))
        _lib.check(lib.mgpt_moe_save_routing(h, saved[-1].data_ptr() + at, stream))
    y = torch.empty_like(x)
    for i, how in enumerate(settings):
        layer.set_routing(**how)
        for j, state in enumerate(saved):
            _lib.check(lib.mgpt_moe_forward_with_routing(h, x.data_ptr(), y.data_ptr(), 100, _lib.IO_BF16, layer._ws.data_ptr(), layer._ws.numel(), state.data_ptr() + at, stream))
            if i == j:
                layer.check_status()
            else:
                with pytest.raises(MoeError, match="saved routing"):
                    layer.check_status()
    layer.set_routing("sigmoid", bias=bias.clone())                     # another tensor, the same setting
    layer.recompute_into(x, y, saved[5][at:at + size] if at % 16 else saved[5][:size])
    layer.check_status()
