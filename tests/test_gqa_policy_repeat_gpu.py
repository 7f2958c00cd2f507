"""Lexical GQA routes repeated on one bank until their hits are many times its
nodes: the hit list of a query starts at its beginning, whatever the queries
before left and whatever the memory held when the bank was made."""

import numpy as np
import pytest

import oracle as O
from graftrepository_b200.cuda_router import CudaGQARouteSidecar

pytestmark = pytest.mark.gpu


def test_hits_of_many_queries_do_not_add_up():
    n, kv, d, h = 96, 2, 64, 4
    rng = np.random.default_rng(3)
    counts = rng.integers(1, 20, n)
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint64)
    keys = O.f32_to_bf16_bits(rng.standard_normal(int(off[-1]) * kv * d).astype(np.float32))
    lex = [["all"] + (["odd"] if i % 2 else []) for i in range(n)]
    bank = CudaGQARouteSidecar(device=0).create_bank_csr(keys.view(np.uint16), off, kv, d)
    bank.set_route_policy(lexical_keys=lex)
    qs = rng.standard_normal((2, h, 1, d)).astype(np.float32)
    qlex = [["all"], ["odd", "absent"]]
    want = [O.gqa_route_policy(keys, off, kv, d, q, 5, node_lexical=lex, query_lexical=x)
            for q, x in zip(qs, qlex)]
    for _ in range(40):  # 40 x 144 hits on 96 nodes
        ids, scores = bank.route_policy_topk(qs, topk=5, lexical_keys=qlex)
        for i, (want_ids, want_scores) in enumerate(want):
            assert np.array_equal(ids[i], want_ids) and np.array_equal(scores[i], want_scores), i
    bank.close()
