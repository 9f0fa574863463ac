"""Layers that keep their inputs as 8-bit records and multiply in 4-bit blocks (B200 only). Every stage is checked on
the inputs that the device itself produced for it, so the tolerances stay those of a single kernel."""
import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU
from nervanagpu_b200 import convnet_benchmarks as cb
from nervanagpu_b200.layers import ConvLayer, FullLayer, PoolLayer, link_records
from oracle import reference_math as rm
from tests._util import assert_close, f32_tol, rn16_tol
from tests.test_blocks_gpu import product_tol

pytestmark = pytest.mark.gpu
f32 = np.float32


def chain(ng, **kwargs):
    confs = [cb._data(64, 8, 8), cb._conv(16, 3, pad=1), cb._conv(24, 3, pad=1), cb._pool(2, 2), cb._full(72), cb._full(40)]
    return cb.build_network(ng, confs, seed=5, **kwargs)


def test_link_records_says_what_can_be_shared():
    ng = NervanaGPU(stochastic_round=False)
    layers = chain(ng, checkpoint=True)
    data, c1, c2, pool, f1, f2 = layers
    assert [l.checkpoint for l in layers] == [False, False, True, False, True, True]
    assert [l.masked_above for l in layers] == [False, True, False, False, True, False]
    assert [l.masks_below for l in layers] == [False, False, True, False, False, True]
    assert link_records(layers) == [False, True, False, True, True, False]
    assert c1.fprop_out.ptr == f1.fprop_out.ptr != pool.fprop_out.ptr       # two buffers in turn
    plain = chain(ng)
    assert not any(l.masked_above or l.masks_below for l in plain) and len({l.fprop_out.ptr for l in plain}) == 6


@pytest.mark.parametrize("products", [None, "mxfp4", "nvfp4"])
def test_chain_with_records_and_4_bit_products(products):
    ng = NervanaGPU(stochastic_round=False)
    data, c1, c2, pool, f1, f2 = layers = chain(ng, checkpoint=True, products=products)
    lr = -0.05
    for l in layers:
        l.learning_rate = lr
    acts, x = {}, None
    for l in layers:
        x = l.fprop(x)
        acts[l] = x.get()                       # (the buffer may be another layer's output later)
    W = {l: l.weights.get() for l in (c1, c2, f1, f2)}
    below = {c2: acts[c1], f1: acts[pool], f2: acts[f1]}
    record = {}
    for l, a in below.items():
        a2 = a.reshape(l.dimI2)
        got = ng.dequantize(l.record, ng.empty(l.dimI2)).get()
        assert np.array_equal(got, rm.block_values(a2, "mxfp8").astype(np.float16)) and (got > 0).any()
        assert np.array_equal(got > 0, a2 > 0)
        record[l] = got
    for l in (f1, f2):
        X = below[l].reshape(l.dimI)
        if products:
            ws, xs = l.scales if products == "nvfp4" else (1.0, 1.0)
            a, b = rm.block_values(W[l], products, 1, ws), rm.block_values(X, products, 0, xs)
        else:
            a, b = W[l].astype(np.float64), X.astype(np.float64)
        ref = np.maximum(a @ b, 0)
        assert_close(acts[l], ref, product_tol(ref, np.abs(a) @ np.abs(b), l.nIn), "fprop")
        assert (acts[l] > 0).any()

    rng = np.random.default_rng(9)
    E = (rng.uniform(-1, 1, f2.dimO) * 0.25).astype(np.float16)
    dE = ng.array(E)

    def full_bprop(l, e, out_above):
        """Deltas in (masked already, or by this layer's own output), checked: deltas out, gradient, weights."""
        down = l.bprop(e)
        em = e.get().astype(np.float64)
        w = W[l].astype(np.float64)
        ref, mag = w.T @ em, np.abs(w.T) @ np.abs(em)
        if l.masks_below:
            mask = record[l] > 0
            ref, mag = np.where(mask, ref, 0), np.where(mask, mag, 0)
            assert (down.get()[~mask] == 0).all()
        assert_close(down.get(), ref, product_tol(ref, mag, l.nOut), "deltas")
        xr = record[l].astype(np.float64)
        dw, mag = em @ xr.T, np.abs(em) @ np.abs(xr.T)
        got = l.updat_out.get()
        assert_close(got, dw, product_tol(dw, mag, 64), "gradient")
        want = (W[l].astype(f32) + got.astype(f32) * f32(lr)).astype(np.float16).astype(f32)
        assert_close(l.weights.get(), want, 2.0 ** -10 * np.abs(want) + 1e-6, "weights")
        return down

    d = full_bprop(f2, dE, None)
    assert np.array_equal(dE.get(), np.where(acts[f2] > 0, E, 0))       # the top layer masks by its own output
    before = d.get()
    d = full_bprop(f1, d, f2)
    assert np.array_equal(f2.bprop_out.get(), before)                   # the layer above has masked these
    d = pool.bprop(d)
    e2 = np.where(acts[c2] > 0, d.get().reshape(acts[c2].shape), 0)
    d = c2.bprop(d)                         # no record above it: masks by its own output
    cd = rm.ConvDims(64, 16, 24, 1, 8, 8, 1, 3, 3, 0, 1, 1, 1, 1, 1)
    ref = rm.conv_bprop_fast(cd, W[c2], e2)
    mask = (record[c2] > 0).reshape(ref.shape)
    mag = rm.conv_bprop_fast(cd, np.abs(W[c2].astype(f32)), np.abs(e2.astype(f32)))
    assert (d.get().reshape(ref.shape)[~mask] == 0).all()
    assert_close(d.get().reshape(ref.shape), np.where(mask, ref, 0), rn16_tol(np.where(mask, ref, 0), mag, 9 * 24), "conv deltas")
    X2 = record[c2].reshape(c2.dimI)
    ref = rm.conv_update_fast(cd, X2, e2)
    assert_close(c2.updat_out.get(), ref, f32_tol(rm.conv_update_fast(cd, np.abs(X2.astype(f32)), np.abs(e2.astype(f32))), 64 * 64), "conv dF")
    e1 = d.get()
    c1.bprop(d)
    assert np.array_equal(d.get(), e1)                                  # masked already
    I = data.fprop_out.get()
    cd = rm.ConvDims(64, 8, 16, 1, 8, 8, 1, 3, 3, 0, 1, 1, 1, 1, 1)
    ref = rm.conv_update_fast(cd, I, e1.reshape(c1.dimO))
    mag = rm.conv_update_fast(cd, np.abs(I.astype(f32)), np.abs(e1.reshape(c1.dimO).astype(f32)))
    assert_close(c1.updat_out.get(), ref, f32_tol(mag, 64 * 64), "first conv dF")


def test_fixed_weights_follow_a_descent_and_recorded_steps_repeat():
    ng = NervanaGPU(stochastic_round=False)
    ng.stream = ng.new_stream()
    layer = FullLayer(ng, np.float16, 32, 96, 64, products="mxfp4", checkpoint=True)
    layer.init_activations()
    layer.init_deltas()
    layer.init_weights(rng=np.random.RandomState(1))
    layer.learning_rate = 0.0
    rng = np.random.default_rng(0)
    X, E = ng.empty((96, 32)), ng.empty((64, 32))
    x = np.maximum(rng.standard_normal((96, 32)), 0).astype(np.float16)
    e = rng.standard_normal((64, 32)).astype(np.float16)
    X.set(x), E.set(e)

    def product(w):
        a, b = rm.block_values(w, "mxfp4", 1), rm.block_values(X.get(), "mxfp4", 0)
        ref = np.maximum(a @ b, 0)
        return ref, product_tol(ref, np.abs(a) @ np.abs(b), 96)

    layer.fix_weights()
    assert layer.weights_fixed
    w0 = layer.weights.get()
    layer.weights[:] = layer.weights * 2.0          # fixed: not seen before fix_weights is called again
    assert_close(layer.fprop(X).get(), *product(w0))
    layer.fix_weights()
    assert_close(layer.fprop(X).get(), *product(layer.weights.get()))
    layer.bprop(E)                                  # a descent: quantised in every pass again
    assert not layer.weights_fixed
    layer.weights[:] = layer.weights * 0.5
    assert_close(layer.fprop(X).get(), *product(w0))

    def step():
        layer.fprop(X)
        layer.bprop(E)

    step()
    run = ng.capture(step)
    for seed in (3, 4):
        r = np.random.default_rng(seed)
        X.set(np.maximum(r.standard_normal((96, 32)), 0).astype(np.float16))
        E.set(r.standard_normal((64, 32)).astype(np.float16))
        run.launch()
        ref, tol = product(layer.weights.get())
        assert_close(layer.fprop_out.get(), ref, tol)
        em = np.where(layer.fprop_out.get() > 0, E.get(), 0).astype(np.float64)
        xr = rm.block_values(X.get(), "mxfp8")
        assert_close(layer.updat_out.get(), em @ xr.T, product_tol(em @ xr.T, np.abs(em) @ xr.T, 32))


def test_new_weights_are_quantised_and_a_first_step_can_be_recorded():
    """All that a fully-connected layer's step needs is there before it: no allocation, which a recording refuses. (A
    convolution's workspace grows when it first runs: that is refused in a recording, with records or without.) Weights of
    ones and inputs of powers of two: exact in every format."""
    ng = NervanaGPU(stochastic_round=False)
    ng.stream = ng.new_stream()
    full = FullLayer(ng, np.float16, 32, 96, 64, products="mxfp4", checkpoint=True)
    full.init_activations()
    full.init_deltas()
    full.init_weights(zeros=True)
    full.fix_weights()
    full.init_weights(zeros=True)
    full.weights.fill(1)
    X, E = ng.empty((96, 32)), ng.empty((64, 32))
    X.fill(2), E.fill(1)

    def step():
        full.fprop(X)
        full.bprop(E)

    ng.capture(step).launch()
    assert (full.fprop_out.get() == 192).all() and (full.updat_out.get() == 64).all()


def test_networks_run_through_the_driver_with_records_and_blocks():
    ng = NervanaGPU(stochastic_round=False)
    res = cb.run_network(ng, "Alexnet", loops=1, out=lambda line: None, checkpoint=True, products="nvfp4")
    assert res["total"][0] > 0 and np.isfinite(res["total"][1])


def test_unknown_products_are_refused():
    with pytest.raises(ValueError):
        FullLayer(NervanaGPU(stochastic_round=False), np.float16, 8, 8, 8, products="int4")
