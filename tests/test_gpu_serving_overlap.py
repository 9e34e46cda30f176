"""Outputs of the serving entries that lie in an input are refused before anything runs; side
by side with one they are not.  (A context that only validates arguments, which the other
refusals are tested with, does not compare the key weights' addresses.)"""
import numpy as np
import pytest

import kraken_hip as kh

pytestmark = pytest.mark.gpu

SEQUENCES, WIDTH, TOKENS, HEADS, KV, D, PT, PAGES, STRIDE = 2, 3, 3, 4, 2, 64, 16, 8, 48
ROOM = 1 << 15  # of each buffer: all that these calls could touch lies in one arena


class Arena:
    """Buffers at places of their own in one allocation of zeros."""

    def __init__(self, torch, sizes):
        assert max(sizes.values()) <= ROOM
        self.sizes = sizes
        self.memory = torch.zeros((len(sizes) + 2) * ROOM, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        self.at = {n: self.memory.data_ptr() + (i + 1) * ROOM for i, n in enumerate(sizes)}

    def view(self, name, at=None):
        return kh.KrakenBuffer(at or self.at[name], self.sizes[name])

    def fill(self, name, values):
        torch = pytest.importorskip("torch")
        raw = torch.from_numpy(np.ascontiguousarray(values).view(np.uint8).ravel().copy())
        first = self.at[name] - self.memory.data_ptr()
        self.memory[first:first + raw.numel()] = raw.cuda()
        torch.cuda.synchronize()

    def cache(self):
        return kh.PagedQ8Cache(*[self.view(n) for n in ("keys", "values", "key_scales",
                                                        "value_scales")], PAGES, PT, KV, D)


POOL = {"keys": PAGES * KV * PT * D, "values": PAGES * KV * PT * D, "key_scales": 4 * PAGES * KV,
        "value_scales": 4 * PAGES * KV}


@pytest.mark.parametrize("f16", [False, True])
def test_key_weights(hip_ctx, f16):
    torch = pytest.importorskip("torch")
    arena = Arena(torch, {**POOL, "query": (2 if f16 else 4) * TOKENS * HEADS * D,
                          "table": 4 * SEQUENCES * WIDTH, "starts": 4 * (SEQUENCES + 1),
                          "lengths": 4 * SEQUENCES, "weights": 4 * SEQUENCES * KV * STRIDE})
    arena.fill("table", np.arange(6, dtype=np.int32))
    arena.fill("starts", np.array([0, 1, 3], np.uint32))
    arena.fill("lengths", np.array([40, 33], np.uint32))
    batch = kh.PagedBatch(*[arena.view(n) for n in ("table", "starts", "lengths")], SEQUENCES,
                          WIDTH, TOKENS, 2, STRIDE)
    name = "key_weights_f16q_paged_q8_kv" if f16 else "key_weights_f32_paged_q8_kv"

    def status(at=None):
        return hip_ctx.status(name, arena.view("query"), arena.cache(), batch, HEADS, 0, 0.0,
                              arena.view("weights", at), STRIDE)

    before = arena.memory.clone()
    size = arena.sizes["weights"]
    for other in ("query", "table", "starts", "lengths", "keys", "key_scales"):
        first, end = arena.at[other], arena.at[other] + arena.sizes[other]
        for at in (first, end - 4, first - size + 4):
            assert status(at) == kh.INVALID_ARGUMENT, (other, at - first)
            assert "must not overlap" in kh.last_error()
    torch.cuda.synchronize()
    assert torch.equal(arena.memory, before)
    for at in (arena.at["table"] - size, arena.at["lengths"] + arena.sizes["lengths"], None):
        assert status(at) == kh.OK, kh.last_error()
    w = arena.memory[arena.at["weights"] - arena.memory.data_ptr():][:size].cpu().numpy()
    w = w.view(np.float32).reshape(SEQUENCES, KV, STRIDE)
    # Zero keys weigh alike: two query heads' one from each row.
    np.testing.assert_allclose(w.sum(-1), [[2.0] * KV, [4.0] * KV], rtol=1e-5)


def test_gathered_weights(hip_ctx):
    torch = pytest.importorskip("torch")
    keep, width = 20, 2
    arena = Arena(torch, {**POOL, "table": 4 * SEQUENCES * WIDTH, "kept": 4 * SEQUENCES * KV * keep,
                          "counts": 4 * SEQUENCES, "target": 4 * SEQUENCES * width,
                          "weights": 4 * SEQUENCES * KV * STRIDE,
                          "moved": 4 * SEQUENCES * KV * STRIDE})
    arena.fill("table", np.array([0, 1, 2, 0, 1, 3], np.int32))
    arena.fill("target", np.arange(4, 8, dtype=np.int32))
    arena.fill("counts", np.array([keep, 3], np.uint32))
    arena.fill("kept", np.tile(2 * np.arange(keep, dtype=np.int32), (SEQUENCES, KV, 1)))
    weights = np.arange(SEQUENCES * KV * STRIDE, dtype=np.float32).reshape(SEQUENCES, KV, STRIDE)
    arena.fill("weights", weights)

    def status(at=None):
        v = arena.view
        return hip_ctx.status("gather_kv_pages_q8", arena.cache(), v("table"), WIDTH, v("kept"),
                              v("counts"), keep, SEQUENCES, v("target"), width, v("weights"), STRIDE,
                              v("moved", at))

    before = arena.memory.clone()
    size = arena.sizes["moved"]
    for other in (*POOL, "table", "kept", "counts", "target", "weights"):
        first, end = arena.at[other], arena.at[other] + arena.sizes[other]
        for at in (first, end - 4, first - size + 4):
            assert status(at) == kh.INVALID_ARGUMENT, (other, at - first)
            assert "must not overlap" in kh.last_error()
    torch.cuda.synchronize()
    assert torch.equal(arena.memory, before)
    for at in (arena.at["key_scales"] - size, arena.at["values"] + arena.sizes["values"], None):
        assert status(at) == kh.OK, kh.last_error()
    got = arena.memory[arena.at["moved"] - arena.memory.data_ptr():][:size].cpu().numpy()
    got = got.view(np.float32).reshape(weights.shape)
    np.testing.assert_array_equal(got[0, :, :keep], weights[0, :, :2 * keep:2])
    np.testing.assert_array_equal(got[1, :, :3], weights[1, :, :6:2])
    assert (got[0, :, keep:] == 0).all() and (got[1, :, 3:] == 0).all()
