"""Log probabilities, entropies and most likely tokens (wl_token_logprobs) against 64 bits; bounds in
tests/serving_ref.py."""
import numpy as np
import pytest

from windlass_amd import hip, paged

from .serving_ref import Logprobs

pytestmark = pytest.mark.gpu


def logits(rng, R, V, spread=2.5):
    z = spread * rng.standard_normal((R, V))
    z[np.arange(R)[:, None], rng.integers(0, V, (R, 3))] += 9.0
    return z


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("V,n_top", [(1, 1), (2, 2), (5, 0), (7, 7), (32, 32), (63, 5), (64, 32), (65, 20), (513, 1), (2047, 20),
                                     (2048, 32), (2049, 5), (2055, 31), (4103, 32), (16384, 20), (50001, 32), (154880, 20)])
def test_rows(gpu, V, n_top, t):
    rng = np.random.default_rng(V)
    R = 3 if V > 20000 else 9
    x = Logprobs(logits(rng, R, V), t, rng.integers(0, V, R), n_top=n_top).run()
    x.check()
    assert x.status() == 0


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("pad,off", [(0, 1), (1, 0), (3, 5), (8, 0), (13, 7), (2, 3)])
@pytest.mark.parametrize("V", [4, 9, 3001])
def test_alignment_and_strides(gpu, V, pad, off, t):
    """Rows that begin anywhere in 16 bytes: their first and last values are read one by one."""
    rng = np.random.default_rng(V + pad)
    Logprobs(logits(rng, 17, V), t, rng.integers(0, V, 17), n_top=min(V, 11), pad=pad, off=off).run().check()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("R,V", [(1, 100003), (40, 9000), (700, 3000), (4097, 130), (5000, 2100)])
def test_few_and_many_rows(gpu, R, V, t):
    """A row in many parts, in a few and in one."""
    rng = np.random.default_rng(R)
    Logprobs(logits(rng, R, V), t, rng.integers(0, V, R), n_top=5).run().check()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n_top", [0, 1, 8])
@pytest.mark.parametrize("entropy", [False, True])
def test_tokens_of_shared_rows(gpu, t, n_top, entropy):
    """The drafted nodes of trees, several to a parent's row; some rows without any."""
    rng = np.random.default_rng(4)
    row = rng.integers(0, 20, 333)
    Logprobs(logits(rng, 20, 5000), t, rng.integers(0, 5000, 333), row, n_top=n_top, entropy=entropy).run().check()


def test_no_tokens_or_nothing_else(gpu):
    rng = np.random.default_rng(5)
    Logprobs(logits(rng, 3, 777), "bf16", [], n_top=4).run().check()
    Logprobs(logits(rng, 3, 777), "f32", [], n_top=0).run().check()
    Logprobs(logits(rng, 3, 777), "f32", [], n_top=0, entropy=False).run().check()
    Logprobs(logits(rng, 3, 777), "f32", [5, 6], n_top=0, entropy=False).run().check()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["equal", "few", "rising", "falling", "blocks", "zeros", "late"])
def test_order_among_equal_and_sorted_values(gpu, what, t):
    """Equal values by id; orders that let everything pass the running bound, or nothing."""
    rng = np.random.default_rng(6)
    R, V = 4, 9001
    z = {"equal": np.full((R, V), 1.25), "few": rng.integers(0, 3, (R, V)).astype(float),
         "rising": np.tile(np.arange(V) * 2.0 ** -6, (R, 1)), "falling": np.tile(-np.arange(V) * 2.0 ** -6, (R, 1)),
         "blocks": np.repeat(rng.standard_normal((R, V // 7 + 1)), 7, 1)[:, :V],
         "zeros": np.where(rng.random((R, V)) < 0.5, 0.0, -0.0), "late": np.where(np.arange(V) >= V - 40, 3.0, 0.0) * np.ones((R, 1))}
    for n_top in (1, 20, 32):
        Logprobs(z[what], t, rng.integers(0, V, R), n_top=n_top).run().check()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 7000])
def test_masked_values(gpu, V, t):
    """-infinity and the type's lowest value where tokens may not come: most of a row, all but one, all."""
    rng = np.random.default_rng(7)
    lowest = float(np.float32(-3.3895314e38 if t == "bf16" else -3.4028235e38))
    z = np.repeat(logits(rng, 1, V), 8, 0)
    z[0, V // 2:] = -np.inf
    z[1, V // 2:] = lowest
    z[2] = np.where(np.arange(V) == V - 3, z[2], -np.inf)
    z[3] = np.where(np.arange(V) == 2, z[3], lowest)
    z[4] = -np.inf
    z[5] = lowest
    z[6] = np.where(np.arange(V) % 2, -np.inf, lowest)
    z[7] = np.where(np.arange(V) % 3 == 1, z[7], -np.inf)
    x = Logprobs(z, t, [1, 1, V - 3, 2, 1, 1, 2, 1], n_top=16).run()
    x.check()
    assert x.get("logp", 8)[2] == 0.0 and x.get("entropy", 8)[2] == 0.0
    Logprobs(z, t, [V - 1] * 8, n_top=3).run().check()  # masked tokens: -infinity, far below


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_values_that_are_not_finite(gpu, value, t):
    """They spoil their own row; the ids are by order all the same."""
    rng = np.random.default_rng(8)
    for V in (50, 6000):
        z = logits(rng, 5, V)
        z[1, V - 7], z[3, 3], z[3, V // 2] = value, value, value
        Logprobs(z, t, [4] * 5, n_top=6).run().check()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("shift,spread", [(1e4, 2.0), (-3e4, 30.0), (0.0, 500.0), (0.0, 1e-3), (3e38, 1e36)])
def test_magnitudes(gpu, shift, spread, t):
    """What is far from zero costs nothing: only differences enter."""
    rng = np.random.default_rng(9)
    Logprobs(shift + spread * rng.standard_normal((6, 5000)), t, rng.integers(0, 5000, 6), n_top=5).run().check()


def test_tokens_and_rows_outside(gpu):
    rng = np.random.default_rng(10)
    x = Logprobs(logits(rng, 4, 300), "bf16", [5, -2, 300, 7, 299, 2 ** 31 - 1], [0, 1, 2, -1, 3, 4], n_top=2)
    x.run()
    assert x.status() == paged.E_SLOT
    got = x.get("logp", 6)
    assert np.isnan(got[[1, 2, 3, 5]]).all() and np.isfinite(got[[0, 4]]).all()
    x.token, x.row = [5, 0, 0, 0, 299, 0], [0, 0, 0, 0, 3, 0]
    x.check(bad_tokens=(1, 2, 3, 5))


def test_places_without_a_token(gpu):
    """Token -1, whatever its row: nothing is written and nothing is wrong."""
    rng = np.random.default_rng(11)
    x = Logprobs(logits(rng, 3, 500), "f32", [5, -1, 7, -1, -1], [0, 1, 2, -1, 99], n_top=4).run()
    assert x.status() == 0
    got = x.get("logp", 5)
    assert (got[[1, 3, 4]] == x.fill).all()
    Logprobs(x.z, "f32", [5, 7], [0, 2], n_top=4).run().check()
    assert np.array_equal(got[[0, 2]], Logprobs(x.z, "f32", [5, 7], [0, 2]).run().get("logp", 2))


def test_offsets_past_32_bits(gpu):
    """Rows behind the first 4 GiB of the logits: strides of 2^24 elements."""
    R, V, stride = 300, 100, 1 << 24
    rng = np.random.default_rng(11)
    z = logits(rng, R, V)
    x = Logprobs(z, "bf16", rng.integers(0, V, R), n_top=3)
    big = hip.DeviceBuffer(2 * (stride * (R - 1) + V))
    from .paged_ref import bf16_bits
    for r in range(R):
        big.upload(bf16_bits(x.z[r]), 2 * stride * r)
    x.args.d_logits, x.args.stride = big.ptr, stride
    x.run().check()
    big.free()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("V", [33, 700, 2100, 8000, 17000, 70000])
def test_rows_of_few_values(gpu, V, t):
    """Many values reach the bound of the most likely: the lists run full, or the row is read again."""
    rng = np.random.default_rng(V)
    z = np.stack([np.full(V, -2.0), rng.integers(0, 2, V).astype(float), np.where(rng.random(V) < 0.03, 4.0, rng.standard_normal(V)),
                  np.where(np.arange(V) < V // 2, 1.0, 0.0)])
    for n_top in (1, 32):
        Logprobs(z, t, rng.integers(0, V, 4), n_top=n_top).run().check()


def fastest(x, times=12):
    """The shortest of some calls, in ms."""
    stream, a, b, t = hip.Stream(), hip.Event(), hip.Event(), []
    for _ in range(times):
        a.record(stream)
        paged.token_logprobs(x.args, stream.handle)
        b.record(stream)
        b.synchronize()
        t.append(a.elapsed_ms(b))
    stream.destroy()
    return min(t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_a_list_of_equal_values_is_cut_once(gpu, t):
    """Where a grammar leaves fewer values than are asked for, the others are equal: -infinity. The row is then read again
    by one work-group (some 5 times the usual row's time); with a list that runs full at every step it is some 100."""
    rng = np.random.default_rng(12)
    V = 262144
    z = logits(rng, 1, V)
    usual = Logprobs(z, t, [5], n_top=20).run()
    for few in (np.where(np.arange(V) % 30001 == 7, z, -np.inf), np.full((1, V), 0.5), np.where(np.arange(V) > V - 9, z, -1e30)):
        x = Logprobs(few, t, [7], n_top=20).run()
        x.check()
        assert fastest(x) < 25 * fastest(usual)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("R,V", [(1, 163839), (1, 163841), (2, 200003), (3, 262144), (1, 1 << 20)])
def test_large_vocabularies(gpu, R, V, t):
    """More lanes of a row than the second launch's threads hold the largest values of; some of the most likely in the
    last parts, all of them, and as many as are asked for beside equal ones."""
    rng = np.random.default_rng(V)
    z = logits(rng, R, V)
    late = z.copy()
    late[:, V - 3000:] += 8.0
    ties = np.round(2 * z) / 2
    ties[:, V - 40:] = ties.max(1, keepdims=True)
    for x in (z, late, ties):
        for n_top in (1, 32):
            Logprobs(x, t, rng.integers(0, V, R), n_top=n_top).run().check()
