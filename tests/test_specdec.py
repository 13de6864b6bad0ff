"""CPU side of the speculative-decoding operators: the plain implementations
that the GPU tests compare with, held to the host allocator and to closed
forms, and the refusals of the calls that need no pool."""
import ctypes

import numpy as np
import pytest
import torch

import pagedkv
from pagedkv import _lib
import specdec_ref as ref


def test_reference_step_tables_is_the_host_allocator():
    rng = np.random.default_rng(3)
    bs, nb, n, width = 4, 200, 6, 24
    alloc = pagedkv.BlockAllocator(nb, bs)
    tables = [pagedkv.BlockTable() for _ in range(n)]
    seq = np.zeros(n, np.int64)
    have, dev = np.zeros(n, np.int64), np.zeros((n, width), np.int64)
    free, count = np.arange(nb - 1, -1, -1), nb  # BlockAllocator::new's free list
    for _ in range(6):
        new = rng.integers(0, 12, n)
        r = ref.step_tables(seq, new, dev, have, free, count, bs, nb, 100)
        assert r["status"][0] == 0
        want = []
        for i in range(n):
            alloc.ensure_capacity(tables[i], int(seq[i] + new[i]))
            assert tables[i].blocks == list(r["block_tables"][i][:r["n_blocks"][i]])
            want += [alloc.slot(tables[i], int(seq[i]) + t) for t in range(new[i])]
        assert alloc.free_count() == r["free_count"][0]
        assert list(r["slot_mapping"][:len(want)]) == want
        seq, have, dev, count = seq + new, r["n_blocks"], r["block_tables"], int(r["free_count"][0])


def test_reference_verification_keeps_the_target_distribution():
    # over many draws the first token of a request with one draft is
    # distributed as p, whatever q is (the point of the scheme).  A count over n
    # draws is off by at most 5 sqrt(p (1 - p) n) with probability above 1 - 6e-7.
    rng = np.random.default_rng(5)
    v, n = 5, 20000
    logits = rng.normal(size=(1, v)) * 1.5
    draft = rng.normal(size=(1, v)) * 1.5
    p = np.exp(logits[0]) / np.exp(logits[0]).sum()
    q = np.exp(draft[0]) / np.exp(draft[0]).sum()
    cu = list(range(n + 1))
    d = rng.choice(v, n, p=q)
    tok, acc = ref.verify(np.repeat(logits, 2 * n, 0), d, cu, rng.random(n), rng.random(n),
                          np.repeat(draft, n, 0), np.ones(n))
    first = tok[2 * np.arange(n)]
    for t in range(v):
        assert abs((first == t).sum() - n * p[t]) <= 5 * np.sqrt(n * p[t] * (1 - p[t]))


def test_reference_sparse_attention_over_all_blocks_is_attention():
    rng = np.random.default_rng(7)
    k, v = rng.normal(size=(2, 6, 4, 2, 8))
    q = rng.normal(size=(1, 4, 8))
    tables, ctx = np.array([[3, 1, 5]]), [10]
    out, _ = ref.sparse_attention(q, k, v, np.tile(np.arange(3), (1, 2, 1)), tables, None, ctx, 4, 0.3)
    kk, vv = (x[tables[0]].reshape(12, 2, 8)[:10] for x in (k, v))
    for h in range(4):
        s = 0.3 * kk[:, h // 2] @ q[0, h]
        w = np.exp(s) / np.exp(s).sum()
        assert np.allclose(out[0, h], w @ vv[:, h // 2], atol=1e-14)


# -- refusals that need no GPU: status and message, nothing enqueued ------------
def _buffers(n):
    """n disjoint, aligned, never dereferenced addresses 1 MiB apart."""
    return [(i + 1) << 20 for i in range(n)]


def _step(**over):
    b = _buffers(14)
    a = dict(block_size=16, num_blocks=100, seq_lens=b[0], new_lens=b[1], n_seqs=4,
             block_tables=b[2], n_blocks=b[3], max_blocks_per_seq=8, free_list=b[4], free_len=50,
             free_count=b[5], max_tokens=32, block_tables_out=b[6], n_blocks_out=b[7],
             free_count_out=b[8], context_lens=b[9], cu_q_lens=b[10], positions=b[11],
             slot_mapping=b[12], status=b[13], stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return pagedkv.lib().pkv_step_tables(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(block_size=24), _lib.PKV_ERR_UNSUPPORTED), (dict(block_size=0), _lib.PKV_ERR_UNSUPPORTED),
    (dict(block_size=512), _lib.PKV_ERR_UNSUPPORTED), (dict(num_blocks=0), _lib.PKV_ERR_INVALID),
    (dict(n_seqs=-1), _lib.PKV_ERR_INVALID), (dict(max_blocks_per_seq=0), _lib.PKV_ERR_INVALID),
    (dict(free_len=-1), _lib.PKV_ERR_INVALID), (dict(max_tokens=-1), _lib.PKV_ERR_INVALID),
    (dict(num_blocks=1 << 27), _lib.PKV_ERR_INVALID),
    (dict(max_blocks_per_seq=1 << 27), _lib.PKV_ERR_INVALID),
    (dict(seq_lens=None), _lib.PKV_ERR_INVALID), (dict(free_count=None), _lib.PKV_ERR_INVALID),
    (dict(free_list=None), _lib.PKV_ERR_INVALID), (dict(status=None), _lib.PKV_ERR_INVALID),
    (dict(slot_mapping=None), _lib.PKV_ERR_INVALID), (dict(seq_lens=2), _lib.PKV_ERR_INVALID),
    # outputs over inputs that other workgroups read, or over each other
    (dict(n_blocks_out=4 << 20), _lib.PKV_ERR_INVALID),
    (dict(free_count_out=6 << 20), _lib.PKV_ERR_INVALID),
    (dict(context_lens=1 << 20), _lib.PKV_ERR_INVALID),
    (dict(block_tables_out=(3 << 20) + 4), _lib.PKV_ERR_INVALID),
    (dict(positions=13 << 20), _lib.PKV_ERR_INVALID),
])
def test_step_tables_refuses(over, code):
    assert _step(**over) == code
    assert pagedkv.lib().pkv_last_error(None)


def _verify(**over):
    b = _buffers(10)
    a = dict(target_logits=b[0], target_dtype=pagedkv.BF16, target_row_stride=100,
             draft_logits=b[1], draft_dtype=pagedkv.F32, draft_row_stride=100, draft_tokens=b[2],
             cu_drafts=b[3], batch=3, total_drafts=6, vocab=100, uniforms=b[4], final_uniforms=b[5],
             temperatures=b[6], out_tokens=b[7], n_accepted=b[8], workspace=b[9],
             workspace_bytes=1 << 20, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return pagedkv.lib().pkv_verify_drafts(*a.values())


@pytest.mark.parametrize("over", [
    dict(batch=-1), dict(total_drafts=-1), dict(vocab=0), dict(vocab=1 << 24),
    dict(target_dtype=7), dict(draft_dtype=-1), dict(target_logits=None), dict(cu_drafts=None),
    dict(draft_tokens=None), dict(uniforms=None), dict(final_uniforms=None),
    dict(out_tokens=None), dict(n_accepted=None), dict(target_row_stride=99),
    dict(draft_row_stride=99), dict(target_logits=1), dict(draft_logits=2), dict(uniforms=2),
    dict(workspace=None), dict(workspace_bytes=100), dict(workspace=8 + (1 << 20)),
    dict(batch=1 << 30),
])
def test_verify_drafts_refuses(over):
    assert _verify(**over) == _lib.PKV_ERR_INVALID
    assert pagedkv.lib().pkv_last_error(None)


@pytest.mark.parametrize("over", [
    # workgroups of a request read what another of them would write
    dict(out_tokens=3 << 20), dict(out_tokens=(3 << 20) - 32), dict(out_tokens=(3 << 20) + 20),
    dict(n_accepted=4 << 20), dict(n_accepted=(5 << 20) + 20), dict(out_tokens=(6 << 20) + 8),
    dict(n_accepted=7 << 20), dict(n_accepted=8 << 20), dict(workspace=8 << 20),
    dict(workspace=(9 << 20) - 16), dict(workspace=1 << 20), dict(workspace=2 << 20),
    # rows of logits: the last one's last elements, and any row of a strided array
    dict(n_accepted=(1 << 20) + 9 * 200 - 4), dict(out_tokens=(2 << 20) + 6 * 400 - 4),
    dict(target_row_stride=120, n_accepted=(1 << 20) + 240 * 3 - 4),
    dict(target_row_stride=120, n_accepted=(1 << 20) + 240 * 3 + 196),
    dict(target_row_stride=101, out_tokens=(1 << 20) + 200),
])
def test_verify_drafts_refuses_overlapping_arrays(over):
    assert _verify(**over) == _lib.PKV_ERR_INVALID
    assert b"overlap" in pagedkv.lib().pkv_last_error(None)


def test_empty_calls_and_queries():
    L = pagedkv.lib()
    assert _verify(batch=0) == 0
    assert L.pkv_verify_workspace_bytes(0, 0, 100, 0) == 0
    assert L.pkv_verify_workspace_bytes(30, 600, 100, 1) > \
        L.pkv_verify_workspace_bytes(30, 600, 100, 0) > 0
    assert L.pkv_key_bounds_bytes(None) == 0
    assert L.pkv_select_workspace_bytes(None, 1, 1, 1, 1, 1, 1) == 0
    assert L.pkv_sparse_workspace_bytes(None, 1, 1, 1) == 0
    for name in ("pkv_key_bounds", "pkv_select_blocks", "pkv_sparse_attention"):
        fn = getattr(L, name)
        args = [None] + [0 if t in (ctypes.c_int, ctypes.c_size_t) else 0.0 if t is ctypes.c_float
                         else None for t in fn.argtypes[1:]]
        assert fn(*args) == _lib.PKV_ERR_INVALID, name


def test_verify_workspace_query_has_the_calls_limits():
    query, most = pagedkv.lib().pkv_verify_workspace_bytes, 1 << 29
    # (drafts and their rows: 3 2^29 rows still count in 32 bits)
    assert query(most, most, 1, 1) > query(most, most, 1, 0) > 0
    for batch, drafts in ((1, most + 1), (1, 1 << 30), (most + 1, 0), (1 << 30, 1 << 30)):
        assert query(batch, drafts, 100, 1) == query(batch, drafts, 100, 0) == 0
        assert _verify(batch=batch, total_drafts=drafts) == _lib.PKV_ERR_INVALID


def test_python_refuses_host_tensors():
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        pagedkv.step_tables(z, z, torch.zeros((4, 2), dtype=torch.int32), z, z, z[:1], 16, 10, 5)
    with pytest.raises(ValueError):
        pagedkv.verify_drafts(torch.zeros((5, 10)), z, z[:2], torch.zeros(4), torch.zeros(1))
