"""The cache of quantised weights answers for the tensor that it quantised, not for another one that has taken its place."""
import torch

from deep_ep.ops.fp8_training import Fp8WeightCache, block_quant


def test_a_new_tensor_in_the_memory_of_a_freed_one():
    """Same address, version and (CPython uses freed objects again) the same `id`, other values."""
    memory = bytearray(2 * 128 * 128 * 2)
    cache, seen = Fp8WeightCache(), set()
    for value in range(1, 40):
        w = torch.frombuffer(memory, dtype=torch.bfloat16).view(2, 128, 128)
        torch.frombuffer(memory, dtype=torch.bfloat16).fill_(value)
        again = (id(w), w._version, w.data_ptr()) in seen
        seen.add((id(w), w._version, w.data_ptr()))
        got, want = cache.get(w), block_quant(w, transposed=True)
        assert all(torch.equal(g.view(torch.uint8), v.view(torch.uint8)) for g, v in zip(got, want)), again
        assert cache.get(w)[0] is got[0]
        del w
