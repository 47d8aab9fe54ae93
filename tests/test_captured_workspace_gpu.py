"""Workspaces of the matmuls that a stream first needs while a graph is captured on it."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture
def new_context(kt, monkeypatch):
    """A context without workspaces, and free device memory full of ones for those to come."""
    from kotensor_b200.quantized import Context
    monkeypatch.setattr(Context, "_by_device", {})
    torch.cuda.synchronize()
    ones = torch.full((256 << 20,), 0xFF, dtype=torch.uint8, device="cuda")
    del ones
    torch.cuda.empty_cache()
    return Context.get(0)


@pytest.mark.parametrize("m", [1, 4, 24, 130])
def test_a_graph_does_not_need_an_earlier_ones_replay(oracle, new_context, m):
    from kotensor_b200 import MatMul, Quantization, QuantizedTensor
    rng = np.random.default_rng(m)
    w = QuantizedTensor.quantize(torch.from_numpy(rng.standard_normal((4096, 256), dtype=np.float32)).cuda(), Quantization.INT4)
    x = torch.from_numpy(rng.standard_normal((m, 4096), dtype=np.float32)).cuda()
    outs = [torch.zeros(m, 256, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    graphs, stream = [], torch.cuda.Stream()
    for out in outs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            MatMul.multiply_quantized(x, w, out, m, accumulate=False)
        graphs.append(g)
    graphs[1].replay()  # the first graph has not run
    MatMul.multiply_quantized(x, w, outs[2], m, accumulate=False)
    torch.cuda.synchronize()
    assert torch.equal(outs[1], outs[2])
    for g in graphs * 2:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2]) and new_context.take_error() == 0


def test_drafts_after_a_text_of_one_token(oracle, new_context):
    """generate_batch of one token captures a step that it does not replay; the graph of the drafted passes is captured on
    the same stream after it."""
    from test_decoder_paged_gpu import decoder
    prompts = np.random.default_rng(12).integers(0, 700, (2, 15)).tolist()
    options = dict(max_seq=128, batch=2, kv_bits=16)
    d = decoder("int4_gqa", **options)
    d.generate_batch(prompts, 1)
    d.reset()
    texts = d.generate_drafted(prompts, 40, nodes=12)
    assert texts == decoder("int4_gqa", **options).generate_drafted(prompts, 40, nodes=12)
    assert new_context.take_error() == 0
