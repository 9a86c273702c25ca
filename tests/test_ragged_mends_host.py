"""The ragged decode operators' binding where there is no GPU: buffers of
another device are refused before the library is called, and what is left out
is filled in."""
import pytest

import specdec_b200 as sd


class Stand:
    """What the binding asks of a tensor."""
    is_cuda = True

    def __init__(self, dtype, *shape, device=0):
        self.dtype, self.shape, self.device = "torch." + dtype, shape, device

    def dim(self):
        return len(self.shape)

    def stride(self):
        st, n = [], 1
        for d in reversed(self.shape):
            st.insert(0, n)
            n *= d
        return tuple(st)

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device

    def data_ptr(self):
        return 4096


class Library:
    """Counts calls in place of the compiled one."""
    calls = 0

    def __getattr__(self, name):
        def call(*args):
            Library.calls += 1
            self.args = args
            return 0

        return call


@pytest.fixture
def kv(monkeypatch):
    h = sd.KV8.__new__(sd.KV8)
    h._lib, h.h, h.device = Library(), None, 0
    h.n_heads, h.n_kv_heads, h.head_dim, h.page_tokens, h.block_tokens = 4, 2, 64, 128, 16
    monkeypatch.setattr(sd, "load_library", lambda *a: h._lib)
    Library.calls = 0
    return h


def buffers(**other):
    """The arguments of each call; those named in `other` on another device."""
    i = lambda name, *shape, t="int32": Stand(t, *shape, device=other.get(name, 0))
    layer = sd.KV8Layer(Stand("int8", 3, 2, 128, 64), Stand("int8", 3, 2, 128, 64), Stand("float32", 3, 2, 8),
                        Stand("float32", 3, 2, 8))
    batch = sd.KV8Batch(Stand("int32", 2, 1), Stand("int32", 2), Stand("int32", 3), Stand("int32", 4), Stand("int32", 4),
                        Stand("int64", 4), Stand("int32", 1))
    rows = lambda name, heads: i(name, 4, heads, 64, t="float32")
    return dict(
        plan=(batch, i("held", 2), i("keep", 2), i("q_len", 2), i("ring", 3), i("ring_state", 2), i("ring_state_out", 2)),
        append=(layer, batch, rows("k", 2), rows("v", 2)),
        gather=(layer, i("rows", 4, t="int64"), rows("out_k", 2), rows("out_v", 2)),
        attend=(layer, batch, rows("q", 4), rows("out", 4), i("lse", 4, 4, t="float32")),
        sample=(i("logits", 2, 9, t="float32"), i("u", 2, t="float32"), i("tokens", 2), i("probs", 2, t="float32"),
                i("temperature", 2, t="float32"), i("top_k", 2), i("top_p", 2, t="float32"), i("min_p", 2, t="float32")))


NAMES = dict(plan=["held", "keep", "q_len", "ring", "ring_state", "ring_state_out"], append=["k", "v"],
             gather=["rows", "out_k", "out_v"], attend=["q", "out", "lse"],
             sample=["logits", "u", "tokens", "probs", "temperature", "top_k", "top_p", "min_p"])


@pytest.mark.parametrize("call,name", [(c, n) for c in NAMES for n in NAMES[c]])
def test_a_buffer_of_another_device_is_refused(kv, call, name):
    run = sd.sample if call == "sample" else getattr(kv, call)
    run(*buffers()[call])
    assert Library.calls == 1
    with pytest.raises(ValueError, match="device"):
        run(*buffers(**{name: 1})[call])
    assert Library.calls == 1


@pytest.mark.parametrize("rows,requests,given,passed", [(300, 1, None, 300), (160, 32, None, 5), (64, 64, None, 1), (70, 64, None, 2),
                                                        (0, 3, None, 0), (300, 1, 1, 1), (5, 2, 9, 9)])
def test_rows_of_a_request_that_are_not_given(kv, rows, requests, given, passed):
    # a prompt without max_q must not go the way of single tokens, which reads the cache once for eight rows
    batch = sd.KV8Batch(Stand("int32", requests, 1), Stand("int32", requests), Stand("int32", requests + 1))
    q, out = (Stand("float32", rows, 4, 64) for _ in range(2))
    kv.attend(buffers()["attend"][0], batch, q, out, **({} if given is None else dict(max_q=given)))
    assert kv._lib.args[12] == passed
