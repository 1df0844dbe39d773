"""Mxfp4Dense in the place of a Dense inside the model."""
import pytest
import torch


def _model():
    import gunet_amd as amd
    return amd.GraphUNet(32, out_units=96, depth=3, activation='relu', layer_type='geo_quadrant_gcn', use_bias=True, use_global=True)


def test_the_one_call_forward_wants_float32_layers():
    """The library's whole-model call reads float32 kernels; a model that holds another layer walks its layer objects."""
    import gunet_amd as amd
    model = _model()
    assert model._native_ok()
    for name in ('in_layer', 'out_model'):
        layer = getattr(model, name)
        setattr(model, name, amd.Mxfp4Dense.__new__(amd.Mxfp4Dense))
        assert not model._native_ok(), name
        setattr(model, name, layer)
    assert model._native_ok()


@pytest.mark.gpu
def test_four_bit_layers_inside_the_model(oracle):
    import gunet_amd as amd
    from gpu_helpers import graph_to_dev, make_case, to_dev
    x, graph, _ = make_case(oracle, 20, 24, 0.5)
    model = _model().load_weights(oracle.make_weights(oracle.graph_unet_shapes(), 1), 'cuda')
    x = to_dev(x, torch.float32)
    plain, _ = model(x, graph_to_dev(graph))
    in_layer, out_model = model.in_layer, model.out_model

    seen = []

    class Watched(amd.Mxfp4Dense):
        def __call__(self, x, activation=Ellipsis):
            seen.append(x.clone())
            return super().__call__(x, activation)

    for swap in ('in_layer', 'out_model'):
        model.in_layer, model.out_model = in_layer, out_model
        four = Watched.from_dense(getattr(model, swap))
        setattr(model, swap, four)
        seen.clear()
        y, after = model(x, graph_to_dev(graph))
        assert y.shape == plain.shape and torch.isfinite(y).all() and len(after['edges']) == 4 and len(seen) == 1
        if swap == 'in_layer':
            assert torch.equal(seen[0], x)
        else:
            w4 = amd.mxfp4_quantize(out_model.kernel.t())
            assert torch.equal(y, amd.mxfp4_dense(seen[0], w4))
            assert torch.equal(model.predict(x, graph_to_dev(graph)), amd.mxfp4_dense(seen[0], w4, None, 'relu'))
    model.in_layer, model.out_model = in_layer, out_model
    again, _ = model(x, graph_to_dev(graph))
    assert torch.equal(again, plain)


@pytest.mark.gpu
def test_four_bit_layers_in_a_captured_model(oracle):
    import gunet_amd as amd
    from gpu_helpers import graph_to_dev, make_case, to_dev
    x, graph, _ = make_case(oracle, 20, 24, 0.5)
    model = _model().load_weights(oracle.make_weights(oracle.graph_unet_shapes(), 1), 'cuda')
    model.in_layer, model.out_model = amd.Mxfp4Dense.from_dense(model.in_layer), amd.Mxfp4Dense.from_dense(model.out_model)
    x, dev = to_dev(x, torch.float32), graph_to_dev(graph)
    cap = amd.CapturedForward(model, x, dev)
    for turn in range(4):
        new = x * (1 + turn) if turn % 2 else x.roll(turn, 0)
        got = cap(new).clone()
        want = model.predict(new, {'edge_index': list(dev['edge_index']), 'edges': list(dev['edges']), 'node_loc': dev['node_loc'], 'global': dev['global']})
        torch.cuda.synchronize()
        assert torch.equal(got, want), turn
