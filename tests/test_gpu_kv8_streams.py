"""The layer calls over the 8-bit KV cache on a stream of the caller's, while the
current stream is busy."""
import pytest
import torch

from test_gpu_kv8 import log
from test_gpu_kv8_layer import filled, make_layer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(gpu):
    return make_layer(gpu, 51)


def busy(gpu):
    """Some 20 ms of work on the current stream."""
    a = torch.ones((8192, 8192), dtype=torch.bfloat16, device=gpu)
    for _ in range(20):
        a = (a @ a) * 2.0 ** -13


def test_first_tree_of_a_cache(gpu, layer):
    """The tree's rows are not touched by what the current stream still has to do."""
    from vates_amd.decode import TreeCommit
    from vates_amd.synth import synth_bf16
    log("case: kv8 first tree on a stream")
    P, S, pos0 = 3, 4, 70
    x = synth_bf16(51, 30, (P * S, layer.hidden), device=gpu)
    a, b = (filled(layer, 51, pos0, 160, gpu) for _ in range(2))
    rec = torch.tensor([S, S, S, 1] + [0] * (S + 1), dtype=torch.int32, device=gpu)
    want = layer.tree(x, a, P)
    TreeCommit([a], P, S)(rec, pos0=pos0)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy(gpu)
    got = layer.tree(x, b, P, stream=st)
    torch.cuda.synchronize()
    TreeCommit([b], P, S)(rec, pos0=pos0)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(a.data, b.data)


@pytest.mark.parametrize("bits", [8, 16])
def test_a_prompt_output_is_of_the_call_s_stream(gpu, layer, bits):
    """Memory that the current stream gave up may still be in use there: the output
    of a call on another stream does not take it."""
    from vates_amd.synth import synth_bf16
    log(f"case: prompt output on a stream, {bits} bits")
    x = synth_bf16(51, 31, (40, layer.hidden), device=gpu)
    st = torch.cuda.Stream()
    want = layer.prompt(x, layer.new_cache(64, bits), pos0=0)
    cache = layer.new_cache(64, bits)
    torch.cuda.synchronize()
    given = torch.empty_like(x)
    at = given.data_ptr()
    del given
    got = layer.prompt(x, cache, pos0=0, stream=st)
    torch.cuda.synchronize()
    assert got.data_ptr() != at and torch.equal(got, want)
