"""A decoder layer's projections as a program would run them: QKV on 4-bit weights, heads normed and turned in place, (attention elsewhere,) output projection, norm, SwiGLU
and down projection, norm, eagerly and as one graph."""
import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import ops
from tests import g4_reference as ref
from tests.test_gpu_g4 import Layer
from tests.test_gpu_mx4 import device, done, host, ready

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 5, 40, 260])
def test_a_layer_eagerly_and_as_a_graph(sess, M):
    """Every step against its definition on the step's own input, so that only its own roundings count: sums by sum_bound, results by half a step."""
    rng = np.random.default_rng(M)
    H, D, q_heads, k_heads, F, group = 512, 64, 8, 2, 704, 64
    width = (q_heads + 2 * k_heads) * D
    qkv, o, pair, down = (Layer(sess, rng, n, k, group, gate_up=g, exact=False) for n, k, g in ((width, H, False), (H, q_heads * D, False), (2 * F, H, True), (H, F, False)))
    ws, ws_down = ops.G4Workspace(sess, M, H, 2 * F), ops.G4Workspace(sess, M, F, H)
    bf = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    residual, x, heads, mixed, mid, branch = bf(M, H), bf(M, H), bf(M, width), bf(M, H), bf(M, F), bf(M, H)
    before, streams = bf(M, width), [bf(M, H) for _ in range(2)]
    inv_freq, positions = device((10000.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)), device(np.arange(100, 100 + M).astype(np.int32))
    wq, wk = (device(1 + 0.2 * rng.standard_normal(D)).float() for _ in range(2))
    w1, w2 = (device(1 + 0.2 * rng.standard_normal(H)).float() for _ in range(2))
    y = bf(M, H)

    def step():
        ws.run(qkv.w, x, heads)
        if eager:
            sess.lib.rk_npu_hip_copy(sess.ctx, before.data_ptr(), heads.data_ptr(), before.numel() * 2)
        ops.heads_norm_rotate(sess, heads[:, :q_heads * D].unflatten(1, (q_heads, D)), heads[:, q_heads * D:(q_heads + k_heads) * D].unflatten(1, (k_heads, D)),
                              q_weight=wq, k_weight=wk, positions=positions, inv_freq=inv_freq)
        ws.run(o.w, heads[:, :q_heads * D], mixed) # (the queries in the attention's place)
        ops.block_norm(sess, residual, branch=mixed, weight=w1, stream_out=streams[0], y=y)
        ws.run_swiglu(pair.w, y, mid)
        ws_down.run(down.w, mid, branch)
        ops.block_norm(sess, streams[0], branch=branch, weight=w2, stream_out=streams[1], y=x)

    def fill(seed):
        r = np.random.default_rng(seed)
        residual.copy_(device(r.standard_normal((M, H)), "bf16"))
        x.copy_(device(r.standard_normal((M, H)), "bf16"))
        ready()

    def close(got, want, bound):
        far = np.abs(host(got) - want) - bound - ref.HALF_STEP["bf16"] * (np.abs(want) + bound)
        assert far.max() <= 0, far.max()

    def product(layer, a, K):
        a = host(a)
        return a @ layer.values.T, ref.sum_bound(a, layer.sizes, K) + 2.0 ** -39 * np.abs(a).max(1)[:, None] * layer.sizes.sum(1)[None, :]
    eager = True
    fill(0)
    x0 = x.clone()
    ready()
    step()
    done(sess)
    close(before, *product(qkv, x0, H))
    cut = host(before)[:, :(q_heads + k_heads) * D].reshape(M, -1, D)
    normed = np.concatenate([ref.head_norm(cut[:, :q_heads], host(wq), 1e-6), ref.head_norm(cut[:, q_heads:], host(wk), 1e-6)], axis=1)
    want = ref.rotate(normed, host(positions)[None], host(inv_freq), [0] * (D // 2), False)
    top = 1.4143 * np.abs(want).max(axis=2, keepdims=True)
    close(heads[:, :(q_heads + k_heads) * D], want.reshape(M, -1), (top * (D * 2.0 ** -25 + 12 * 2.0 ** -23) + 0 * want).reshape(M, -1))
    assert torch.equal(heads[:, (q_heads + k_heads) * D:], before[:, (q_heads + k_heads) * D:])
    close(mixed, *product(o, heads[:, :q_heads * D], H))
    s, e = product(pair, y, H)
    silu = ref.silu(s[:, :F])
    close(mid, silu * s[:, F:], 1.1 * e[:, :F] * (np.abs(s[:, F:]) + e[:, F:]) + np.abs(silu) * e[:, F:] + 2.0 ** -19 * np.abs(silu * s[:, F:]) + 1e-30)
    close(branch, *product(down, mid, F))
    eager = False
    fill(1)
    assert sess.lib.rk_npu_hip_capture_begin(sess.ctx) == 0
    step()
    graph = sess.lib.rk_npu_hip_capture_end(sess.ctx)
    assert graph
    for seed in (2, 3, 4):
        fill(seed)
        step()
        done(sess)
        kept = [t.clone() for t in (heads, mixed, mid, branch, *streams, x)]
        fill(seed)
        assert sess.lib.rk_npu_hip_graph_launch(sess.ctx, graph) == 0
        done(sess)
        assert all(torch.equal(a, b) for a, b in zip(kept, (heads, mixed, mid, branch, *streams, x)))
        assert torch.isfinite(x).all()
    sess.lib.rk_npu_hip_graph_free(graph)
    for h in (ws, ws_down, qkv, o, pair, down):
        h.close()
