"""What the calls over a paged cache check on the host before they hand anything to
the library.  No GPU: tensors that say which GPU they are on, and library calls
that are recorded, not made."""
import pytest
import torch

from odiengine_b200 import paged

I32 = torch.int32


class OnGpu:
    """A CPU tensor that passes for one of cuda:`index` (its memory is never followed)."""

    is_cuda = True

    def __init__(self, t, index=0):
        self.t, self.index = t, index

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.index


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(paged, "_call", lambda dev, stream, fn, *args: made.append((fn.__name__, dev, args)))
    return made


def z(*shape, dtype=torch.float32, on=0):
    return OnGpu(torch.zeros(shape, dtype=dtype), on)


def handles(cache=0, tables=0, batch=0, max_pages=4):
    """A cache, tables and a batch of two requests, each on the GPU that is named."""
    c = paged.PagedCache(*(z(6, 2, 16, 64, dtype=torch.float16, on=cache) for _ in range(2)))

    def new(on):
        return paged.PageTables(z(2, max_pages, dtype=I32, on=on), z(2, dtype=I32, on=on), z(6, dtype=I32, on=on), z(1, dtype=I32, on=on), 16)

    return c, new(tables), paged.PagedBatch(new(batch), max_rows=8, max_new=4, heads=4, kv_heads=2)


def step(c, t, b, on=0):
    paged.paged_step(t, b, z(2, dtype=I32, on=on))


def append(c, t, b, on=0):
    paged.qk_rope_append_paged(z(3, 512, on=on), c, b, z(3, 256, dtype=torch.float16, on=on), heads=4, theta=1e4)


def attend(c, t, b, on=0):
    q, out = (z(3, 256, dtype=torch.float16, on=on) for _ in range(2))
    paged.attention_paged(q, c, t, b, out, scale=1.0, scratch=z(64, dtype=torch.uint8, on=on))


def test_handles_of_one_device_go_through(calls):
    for on in (0, 3):
        for op in (step, append, attend):
            op(*handles(on, on, on), on=on)
    assert [dev for _, dev, _ in calls] == [0] * 3 + [3] * 3


@pytest.mark.parametrize("op,where", [(step, dict(batch=1)), (step, dict(tables=1)), (append, dict(batch=1)), (append, dict(cache=1)),
                                      (attend, dict(batch=1)), (attend, dict(tables=1)), (attend, dict(cache=1)),
                                      (attend, dict(tables=1, batch=1))])
def test_handles_of_different_devices_are_refused(calls, op, where):
    """Their addresses would reach a kernel on the other GPU."""
    for on in (0, 1):
        with pytest.raises(ValueError, match="cuda:"):
            op(*handles(**where), on=on)
    assert not calls


def test_a_decoder_refuses_weights_of_another_device():
    from odiengine_b200.decode import ModelWeights

    w = ModelWeights(token_embd=z(10, 4, on=0))
    with pytest.raises(ValueError, match="cuda:1"):
        paged.PagedDecoder(None, w, requests=1, num_pages=1, device="cuda:1")


@pytest.mark.parametrize("logits,starts", [((5,), 3), ((5, 7, 1), 3), ((5, 7), 0), ((5, 7), 1)])
def test_verify_refuses_logits_or_starts_of_no_shape(calls, logits, starts):
    with pytest.raises(ValueError, match="wanted"):
        paged.verify_sampled(z(*logits), z(5, dtype=I32), z(starts, dtype=I32), z(5), z(2), scratch=z(8, dtype=torch.uint8))
    assert not calls
