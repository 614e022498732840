"""examples/decoder.py's captured step at a real vocabulary's size."""
import pytest
import torch
from torch.profiler import ProfilerActivity, profile

from test_gpu_decoder_example import model_and_reference  # noqa: F401

pytestmark = pytest.mark.gpu


def model_of(model_and_reference):  # noqa: F811
    decoder, _ = model_and_reference
    shape = decoder.Shape(layers=1, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=256, vocab=151936)
    return decoder.Decoder(shape, 64)


def test_no_memory_is_set_in_the_capture(cuda, model_and_reference):  # noqa: F811
    """Replays of a recorded memset have given wrong results; torch's argmax over
    as many logits makes one."""
    model = model_of(model_and_reference)
    logits = model.prompt([1, 2, 3])
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        model.decode(logits, 2)
        torch.cuda.synchronize()
    calls = sorted((e.time_range.start, e.name) for e in p.events() if e.name.startswith("hip"))
    names = [name for _, name in calls]
    first, last = names.index("hipStreamBeginCapture"), names.index("hipStreamEndCapture")
    assert first < last and "hipMemsetAsync" not in names[first:last], names[first:last]


def test_every_replay_s_token_is_the_best_of_an_eager_step(cuda, model_and_reference):  # noqa: F811
    a, b = model_of(model_and_reference), model_of(model_and_reference)
    chosen, _ = a.decode(a.prompt([5, 6, 7]), 12)
    logits = b.prompt([5, 6, 7])
    for i, t in enumerate(chosen):
        assert int(logits.argmax()) == t, i
        logits = b.prompt([t])


def test_nothing_to_decode_or_to_read(cuda, model_and_reference):  # noqa: F811
    model = model_of(model_and_reference)
    with pytest.raises(ValueError):
        model.prompt([])
    assert model.decode(model.prompt([4]), 0) == ([], 0.0)
