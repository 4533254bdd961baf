"""How many clusters of blocks of attention over a 4-bit cache a GPU is taken to hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_more_clusters_than_their_blocks_have_places():
    from llm_singularity_b200 import kernels as ops
    ops.prepare(["attention_kv4", "attention_kv4_f32"])
    dev = torch.device("cuda:0")
    for lib, most in (("attention_kv4", 128), ("attention_kv4_f32", 0)):
        for hd in range(32, 257, 32):
            for eights in (1, 2) if hd <= most else (1,):
                blocks = ops._kv4_room(lib, hd, eights, 0, dev)
                clusters = [ops._kv4_room(lib, hd, eights, n, dev) for n in range(2, 9)]
                assert all(0 < n * c <= blocks for n, c in zip(range(2, 9), clusters)), (lib, hd, eights, blocks, clusters)
                assert clusters == sorted(clusters, reverse=True)
    assert ops._kv4_room("attention_kv4", 64, 1, 9, dev) == 0
