"""CPU side of serving from a cache held in 4 bits: the plain implementations that
the GPU tests compare with, held to closed forms, and the refusals of the calls
that need no pool."""
import math

import numpy as np
import pytest
import torch

import pagedkv
from pagedkv import _lib
import serve4_ref as ref


def test_reference_codes_are_the_nearest_of_sixteen():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(50, 64)).astype(np.float16).astype(np.float64)
    c, m, s = ref.quantize(x)
    assert c.min() == 0 and c.max() == 15
    y = x.reshape(50, 2, 32)
    grid = m[..., None] + s[..., None] * np.arange(16)  # every value a group can stand for
    best = np.abs(y[..., None] - grid[:, :, None, :]).min(-1)
    assert np.allclose(np.abs(ref.held(x).reshape(y.shape) - y), best, rtol=0, atol=1e-12)
    # half a step away at most, but for s and m being rounded to f16 (half a step of
    # 2^-11: of s 15 times over, and of m)
    assert np.all(np.abs(ref.held(x).reshape(y.shape) - y)
                  <= (s / 2 + 15 * s * 2 ** -11 + np.abs(m) * 2 ** -11)[..., None])


def test_reference_codes_of_special_groups():
    x = np.zeros((6, 32))
    x[0] = 0.25
    x[1, :3] = (math.nan, math.inf, -math.inf)
    x[2] = np.arange(32) % 16
    x[3] = 1e-9
    x[4, 0] = 70000.0
    x[5] = np.arange(32) * 0.5
    x[5, 31] = 15.0
    h = ref.held(x)
    assert np.all(h[0] == 0.25) and np.array_equal(h[2], x[2])
    assert np.all(h[3] == 0.0)  # below f16's smallest step
    assert np.all(np.isfinite(h)) and h[1, 2] == -65024 and h[4, 0] >= 64960
    # steps of one: halves go to even codes
    assert np.array_equal(h[5], np.clip(np.rint(np.arange(32) * 0.5), 0, 15))


def test_reference_chunk_layout_is_the_headers():
    rng = np.random.default_rng(2)
    hd, bs = 64, 16
    c, m, s = ref.quantize(rng.normal(size=(bs, hd)))
    b = ref.chunk_bytes(True, c, m, s, bs)
    assert b.size == bs * hd * 5 // 8
    w = b[:bs * hd // 2].view(np.uint32).reshape(bs, 4, 2)
    assert (int(w[3, 1, 1]) >> 16) & 15 == c[3, 32 + 8 + 1]  # e = 1 is in the upper half
    assert (int(w[3, 1, 1]) >> 4) & 15 == c[3, 32 + 8 + 2]
    rest = b[bs * hd // 2:].view(np.float16)
    assert rest[(7 // 4 * 2 + 1) * 4 + 7 % 4] == s[7, 1] and rest[bs * 2 + (7 // 4 * 2 + 1) * 4 + 3] == m[7, 1]
    b = ref.chunk_bytes(False, c, m, s, bs)
    v = b[:bs * hd // 2].reshape(bs // 4, 16, 4, 2)
    assert v[9 // 4, 5, 9 % 4, 1] >> 4 == c[9, 5 + 16 * 3]
    assert b[bs * hd // 2:].view(np.float16)[bs * 2 + (7 // 4 * 2 + 1) * 4 + 3] == m[7, 1]


def test_reference_attention_is_a_mean_of_values():
    rng = np.random.default_rng(3)
    q, k, v = rng.normal(size=(2, 4, 8)), rng.normal(size=(6, 2, 8)), rng.normal(size=(6, 2, 8))
    out, a, b, c = ref.attention(q, k, v, 2, 0.0)
    for i, n in ((0, 5), (1, 6)):
        for h in range(4):
            assert np.allclose(out[i, h], v[:n, h // 2].mean(0), atol=1e-15)
    out, _, _, _ = ref.attention(q, k[:1], v[:1], 2, 1.0)
    assert not out[0].any() and np.allclose(out[1, 3], v[0, 1])


def test_reference_logits():
    x = np.array([2.0, -2.0, 1.0, 0.0, -np.inf, 3.0], np.float32)
    got = ref.adjust_logits(x, [0, 1, 1, 4, 9, -1], None, 2, 2.0, 0.5, 0.25, [(5, 1.0), (5, 2.0)], None)
    assert np.array_equal(got, np.float32([1.0, -4.75, 1.0, 0.0, -np.inf, 5.0]))
    got = ref.adjust_logits(x, [], None, 0, 1.0, 0, 0, [], [0b100101])
    assert np.array_equal(got, np.float32([2.0, -np.inf, 1.0, -np.inf, -np.inf, 3.0]))


# -- refusals that need no GPU: status and message, nothing enqueued ------------
def _at(i):
    """Disjoint, aligned, never dereferenced addresses."""
    return (i + 1) << 32


def _prompt(**over):
    a = dict(q=_at(0), k=_at(1), v=_at(2), dtype=1, qs=512, ks=128, vs=128, out=_at(3), out_dtype=1,
             cu_lens=_at(4), n_seqs=2, total=50, max_len=30, n_head=8, n_kv_head=2, head_dim=64,
             scale=0.125, stream=None)
    a.update(over)
    return pagedkv.lib().pkv_prompt_attention(*a.values())


@pytest.mark.parametrize("over", [
    dict(n_seqs=-1), dict(total=-1), dict(dtype=3), dict(out_dtype=2), dict(n_head=7), dict(n_kv_head=0),
    dict(max_len=0), dict(max_len=(1 << 30) + 1), dict(scale=math.nan), dict(scale=-math.inf),
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu_lens=None), dict(q=_at(0) + 8),
    dict(out=_at(3) + 4), dict(cu_lens=_at(4) + 2), dict(qs=511), dict(qs=516), dict(ks=120),
    dict(vs=0), dict(ks=-128), dict(qs=1 << 61), dict(out=_at(0)), dict(out=_at(1) + 16), dict(out=_at(2))])
def test_prompt_attention_refuses(over):
    assert _prompt(**over) == _lib.PKV_ERR_INVALID
    assert b"prompt_attention" in pagedkv.lib().pkv_last_error(None)


def test_prompt_attention_limits():
    assert _prompt(head_dim=96) == _lib.PKV_ERR_UNSUPPORTED
    assert _prompt(n_seqs=1 << 30, total=1 << 12, max_len=1 << 12) == _lib.PKV_ERR_UNSUPPORTED
    assert _prompt(n_seqs=0, q=None) == 0 and _prompt(total=0, out=None) == 0


def _logits(**over):
    a = dict(logits=_at(0), out=_at(1), dtype=2, row_stride=100, out_row_stride=100, batch=4, vocab=100,
             tokens=_at(2), cu_tokens=_at(3), total_tokens=50, prompt_lens=_at(4), repetition=_at(5),
             presence=_at(6), frequency=_at(7), bias_tokens=_at(8), bias_values=_at(9),
             cu_bias=_at(10), total_bias=20, mask=_at(11), n_masks=3, mask_row_words=4,
             mask_rows=_at(12), stream=None)
    a.update(over)
    return pagedkv.lib().pkv_adjust_logits(*a.values())


@pytest.mark.parametrize("over", [
    dict(batch=-1), dict(vocab=0), dict(vocab=1 << 24), dict(dtype=3), dict(total_tokens=-1),
    dict(total_bias=-1), dict(total_tokens=(1 << 30) + 1), dict(total_bias=2 ** 31 - 1), dict(logits=None), dict(out=None), dict(tokens=None), dict(cu_tokens=None),
    dict(bias_tokens=None), dict(bias_values=None), dict(cu_bias=None), dict(row_stride=99),
    dict(out_row_stride=99), dict(logits=_at(0) + 1), dict(out=_at(1) + 1), dict(tokens=_at(2) + 2),
    dict(mask=_at(11) + 1), dict(n_masks=0), dict(mask_row_words=3), dict(mask_rows=None),
    dict(out=_at(0), out_row_stride=101), dict(out=_at(0) + 2), dict(out=_at(2)), dict(out=_at(3)),
    dict(out=_at(9)), dict(out=_at(11)), dict(out=_at(12)), dict(out=_at(5))])
def test_adjust_logits_refuses(over):
    assert _logits(**over) == _lib.PKV_ERR_INVALID
    assert b"adjust_logits" in pagedkv.lib().pkv_last_error(None)
    assert _logits(batch=0, logits=None) == 0


def test_python_refuses_host_tensors():
    z = torch.zeros((4, 8, 64))
    with pytest.raises(ValueError, match="device tensor"):
        pagedkv.prompt_attention(z, z, z, [0, 4])
    with pytest.raises(ValueError, match="device tensor"):
        pagedkv.adjust_logits(torch.zeros((2, 10)))
