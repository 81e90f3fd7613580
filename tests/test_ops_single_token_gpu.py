"""One token, the only number of tokens that is multiplied inside the decoder: the places where its rows,
sub-chunks and chunks end."""

import pytest
import torch

import cuzipnn_b200 as z
from test_ops_gpu import BF, DEV, HF, check_linear, rnd, weight

pytestmark = pytest.mark.gpu

# rows, cols, chunk, sub-chunk bytes: short last chunks and sub-chunks (most segments of the last rounds
# hold nothing), columns that are no multiple of a round, rows over many sub-chunks, over two chunks and
# over many (parts from the middle chunks), rows that end with their chunk, 4 to 64 sub-chunks.
SHAPES = [
    (65, 512, 131072, 8192), (100, 640, 65536, 4096), (100, 640, 65536, 64), (3, 144, 4096, 64), (333, 144, 4096, 256),
    (257, 272, 16000, 1000), (97, 3584, 8192, 512), (40, 20000, 1024, 64), (9, 8192, 8192, 2048), (31, 4096, 131072, 8192),
    (7, 30000, 4096, 1 << 20), (1, 128, 16384, 64), (700, 1280, 16384, 1024), (5, 65552, 8192, 128), (3000, 128, 131072, 8192),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,cols,chunk,sub", SHAPES)
def test_single_token_shapes(rows, cols, chunk, sub, dtype):
    w = rnd(rows, cols, dtype=dtype, scale=0.05, seed=1)
    blob = z.compress_tensor(w, chunk_bytes=chunk, sub_chunk_bytes=sub, min_compress_bytes=0, readback_to_cpu=False)
    check_linear(rnd(1, cols, dtype=dtype), w, blob)


@pytest.mark.parametrize("sub", [64, 256, 1024, 1 << 20])
@pytest.mark.parametrize("chunk", [2048, 65536])
@pytest.mark.parametrize("cols", [640, 7168])
def test_single_token_sub_chunk_counts(cols, chunk, sub):
    w = rnd(100, cols, scale=0.05)
    blob = z.compress_tensor(w, chunk_bytes=chunk, sub_chunk_bytes=sub, min_compress_bytes=0, readback_to_cpu=False)
    check_linear(rnd(1, cols), w, blob)


@pytest.mark.parametrize("kind", ["both", "raw"])
@pytest.mark.parametrize("rows,cols,chunk", [(65, 512, 131072), (333, 144, 4096), (40, 20000, 1024)])
def test_single_token_blob_kinds(kind, rows, cols, chunk):
    """Both planes coded (the second pass of the decoder) and none."""
    w, blob = weight(rows, cols, BF, kind=kind, chunk=chunk)
    check_linear(rnd(1, cols), w, blob)


def test_single_token_at_the_end_of_its_memory():
    """x as the last row of an allocation, where a read past it would leave the tensor."""
    w, blob = weight(65, 512, BF, chunk=131072)
    pool = torch.empty(64 << 20, dtype=BF, device=DEV)
    x = pool[-512:].view(1, 512).copy_(rnd(1, 512))
    check_linear(x, w, blob)


@pytest.mark.parametrize("tokens", [1, 30])
def test_captured_calls_without_gradients(tokens):
    """One graph of a layer and both losses, replayed on other inputs and beside another graph of the
    same calls on a second stream."""
    w, blob = weight(5000, 256, BF, chunk=4096)
    gen = torch.Generator(device=DEV).manual_seed(4)

    def inputs():
        return (torch.randn((tokens, 256), generator=gen, device=DEV).to(BF),
                torch.randint(5000, (tokens,), generator=gen, device=DEV),
                torch.randint(5000, (tokens, 7), generator=gen, device=DEV),
                torch.randn((tokens, 7), generator=gen, device=DEV))

    def step(x, t, ids, logits):
        return [z.blob_linear(x, blob, activation="gelu"), z.blob_cross_entropy(x, blob, t),
                z.blob_distillation(x, blob, logits, ids, temperature=2.0, reduction="none")]

    sets = [inputs() for _ in range(3)]
    want = [step(*s) for s in sets]
    graphs = []
    for _ in range(2):
        held = [v.clone() for v in sets[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        graphs.append((graph, held, out, torch.cuda.Stream()))
    for i in (1, 2, 0, 1):
        torch.cuda.synchronize()
        for j, (graph, held, out, stream) in enumerate(graphs):  # both at once, on different inputs
            with torch.cuda.stream(stream):
                for a, b in zip(held, sets[(i + j) % 3]):
                    a.copy_(b)
                graph.replay()
        torch.cuda.synchronize()
        for j, (_, _, out, _) in enumerate(graphs):
            for a, b in zip(out, want[(i + j) % 3]):
                assert torch.equal(a, b)
