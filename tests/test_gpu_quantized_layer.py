"""The example that runs the 4-bit and 8-bit operators together, against the same layer in 64 bits."""
import numpy as np
import pytest

import lowbits as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompt,page", [(45, 16), (130, 64)])
def test_layer_prompt_and_tokens(hip, prompt, page):
    """Every intermediate is recomputed from the device's own operands (its codes, its pages), so that each output row
    is held to the f32 bounds of its last products: 1e-4 of the row's norm, five times the largest seen in 64 bits
    from f32 scores (2^-24 times some 10^2 of scores' condition)."""
    from demonic_amd.examples.quantized_layer import run
    heads, kv, dim, hidden, steps = 8, 2, 64, 256, 3
    layer, x, out, _, _ = run(hidden=hidden, heads=heads, kv_heads=kv, dim=dim, page=page, prompt=prompt, steps=steps)
    values = []
    for w, s, n, k in ((layer.w_qkv, layer.qkv_scales, layer.wide, hidden), (layer.w_out, layer.out_scales, hidden, heads * dim)):
        qb, sb = hip.mxfp4_row(k)
        values.append(L.mx_values(w.download(np.uint8, (n, qb)), s.download(np.uint8, (n, sb)), k))
    w_qkv, w_out = values
    c = L.Cache(layer.pages, kv, page, dim)
    c.k, c.v = (b.download(np.uint8, a.shape) for b, a in zip(layer.buffers[:2], (c.k, c.v)))
    c.ks, c.vs = (b.download(np.uint8, a.shape) for b, a in zip(layer.buffers[2:], (c.ks, c.vs)))
    table = [layer.table.download(np.int32, (layer.pages,)).tolist()]
    total = prompt + steps
    qx = x.astype(np.float64).copy()
    q, s = L.mx_quantize(x[:prompt])
    qx[:prompt] = L.mx_values(q, s, hidden)
    qkv = qx @ w_qkv.T
    rows = qkv[:, :heads * dim].reshape(total, heads, dim)
    # the last token's pages are the device's at the end: rows that saw other codes then are not held to them
    want, _, _ = c.attend(table, [total], [0, 1], rows[-1:].astype(np.float32), dim ** -0.5)
    y = want.reshape(1, -1) @ w_out.T
    assert np.linalg.norm(out[-1] - y[0]) <= 1e-4 * np.linalg.norm(y[0])
    # the cache holds the tokens' own k and v to 4 bits
    k, v, there = c.tokens(table[0], total)
    assert there.all()
    for got, at in ((k, heads * dim), (v, (heads + kv) * dim)):
        ref = qkv[:, at:at + kv * dim].reshape(total, kv, dim)
        assert np.linalg.norm(got - ref) <= 2.0 ** -4 * np.linalg.norm(ref)
    assert np.isfinite(out).all() and out.shape == (total, hidden)
