"""What stands between the linears, without a GPU: refusals of the C entries before any launch, of the Python calls for tensors that are not
on a GPU, the registered op of a layer with an epilogue, and the way a vLLM layer's bias takes."""
import contextlib
import ctypes as C

import pytest
import torch
from torch._subclasses import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from hygemm_vllm import native, ops, producer
from hygemm_vllm.cache import AttentionCall, Cache, PagedCache, page_bytes

LIBRARY = native.library()
FAKE = 1 << 20   # an address that is never followed: every call below is refused before a launch


def message(status):
    assert status == -1
    return LIBRARY.hg_last_error().decode()


def test_structs_are_the_librarys():
    """Sizes as the compiler lays them out: nine and three pointers, then what the header lists."""
    assert C.sizeof(producer.NormCall) == 9 * 8 + 3 * 8 + 3 * 4 + 3 * 4
    assert C.sizeof(Cache) == 24 and C.sizeof(native.Epilogue) == 32
    assert C.sizeof(AttentionCall) == 8 * 8 + 2 * 8 + 5 * 4 + 4
    assert LIBRARY.hg_cache_page_bytes(16, 128) == page_bytes(16, 128) == 4224 and LIBRARY.hg_cache_page_bytes(48, 64) == page_bytes(48, 64)


def norm(dtype=1, **change):
    fields = dict(x=FAKE, weight=FAKE, codes=FAKE, scales=FAKE, x_stride=256, rows=4, k=256, eps=1e-6, scale=1.0) | change
    return LIBRARY.hg_norm(C.byref(producer.NormCall(**fields)), dtype, None)


@pytest.mark.parametrize("change, text", [
    (dict(k=260), "multiple of 8"), (dict(k=0), "multiple of 8"), (dict(k=32776), "32768"), (dict(rows=-1), "multiple of 8"),
    (dict(k=264), "divisible by 128"), (dict(x=None), "needed"), (dict(weight=None), "needed"), (dict(codes=None, scales=None), "needed"),
    (dict(normed=FAKE), "needed"), (dict(scales=None), "needed"), (dict(residual=FAKE, residual_stride=256), "needs an output"),
    (dict(scale=2.0), "needs an output"), (dict(x=FAKE + 2), "aligned"), (dict(x_stride=260), "aligned"), (dict(weight=FAKE + 8), "aligned"),
    (dict(gate=FAKE + 4, stream_out=FAKE), "aligned"), (dict(residual=FAKE, residual_stride=257, stream_out=FAKE), "aligned"),
])
def test_norm_entry(change, text):
    assert text in message(norm(**change))


def test_norm_entry_dtype_and_nothing_to_do():
    assert "dtype" in message(norm(dtype=2))
    assert "Null" in message(LIBRARY.hg_norm(None, 1, None))
    assert norm(rows=0) == 0


def cache(**change):
    return Cache(**(dict(data=FAKE, pages=4, kv_heads=2, page_size=16, head_dim=64) | change))


BAD_CACHES = [(dict(data=None), "pages and heads"), (dict(pages=0), "pages and heads"), (dict(kv_heads=0), "pages and heads"),
              (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"),
              (dict(page_size=2048), "page_size"), (dict(data=FAKE + 8), "aligned"), (dict(kv_heads=70000), "too many"),
              (dict(pages=1 << 30, page_size=64), "too many")]


@pytest.mark.parametrize("change, text", BAD_CACHES)
def test_a_cache_that_is_none(change, text):
    strides = (C.c_int64 * 4)(128, 64, 128, 64)
    c = C.byref(cache(**change))
    assert text in message(LIBRARY.hg_cache_write(c, FAKE, FAKE, strides, FAKE, 1, 1, None))
    assert text in message(LIBRARY.hg_cache_read(c, FAKE, FAKE, FAKE, 1, 1, None))
    assert text in message(LIBRARY.hg_attention_workspace(c, 1, 2, 1, 0))
    assert text in message(LIBRARY.hg_attention(c, C.byref(attention()), 1, None))


def test_cache_entries():
    strides = (C.c_int64 * 4)(128, 64, 128, 64)
    c = C.byref(cache())
    assert "invalid" in message(LIBRARY.hg_cache_write(c, FAKE, FAKE, strides, FAKE, -1, 1, None))
    assert "invalid" in message(LIBRARY.hg_cache_read(c, FAKE, FAKE, FAKE, 1, 7, None))
    assert "Null" in message(LIBRARY.hg_cache_write(c, None, FAKE, strides, FAKE, 1, 1, None))
    assert "Null" in message(LIBRARY.hg_cache_write(c, FAKE, FAKE, None, FAKE, 1, 1, None))
    assert "aligned" in message(LIBRARY.hg_cache_write(c, FAKE + 4, FAKE, strides, FAKE, 1, 1, None))
    assert "strides" in message(LIBRARY.hg_cache_write(c, FAKE, FAKE, (C.c_int64 * 4)(128, 64, 126, 64), FAKE, 1, 1, None))
    assert "Null" in message(LIBRARY.hg_cache_read(c, FAKE, FAKE, None, 1, 1, None))
    assert "aligned" in message(LIBRARY.hg_cache_read(c, FAKE, FAKE + 8, FAKE, 1, 1, None))
    assert LIBRARY.hg_cache_write(c, None, None, strides, None, 0, 1, None) == 0 and LIBRARY.hg_cache_read(c, None, None, None, 0, 1, None) == 0


def attention(**change):
    fields = dict(q=FAKE, table=FAKE, lengths=FAKE, out=FAKE, q_stride=256, table_stride=4, seqs=2, heads=4, table_width=4, scale=0.1)
    return AttentionCall(**(fields | change))


@pytest.mark.parametrize("change, text", [
    (dict(heads=3), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"), (dict(seqs=-1), "multiple of kv_heads"),
    (dict(table_width=-1), "table width"), (dict(window=-1), "table width"), (dict(table_width=1 << 27), "table width"),
    (dict(seqs=1 << 25), "too much work"), (dict(q=None), "needed"), (dict(lengths=None), "needed"), (dict(table=None), "needed"), (dict(out=None), "needed"),
    (dict(codes=FAKE, scales=FAKE), "needed"), (dict(out=None, codes=FAKE), "needed"), (dict(q=FAKE + 8), "aligned"),
    (dict(q_stride=260), "aligned"), (dict(out=FAKE + 2), "aligned"), (dict(seqs=300, table_width=64), "workspace is needed"),
    (dict(seqs=300, table_width=64, workspace=FAKE + 8), "aligned"),
])
def test_attention_entry(change, text):
    assert text in message(LIBRARY.hg_attention(C.byref(cache()), C.byref(attention(**change)), 1, None))


def test_attention_entry_more():
    one = Cache(data=FAKE, pages=4, kv_heads=1, page_size=16, head_dim=64)
    assert "divisible by 128" in message(LIBRARY.hg_attention(C.byref(one), C.byref(attention(heads=3, out=None, codes=FAKE, scales=FAKE)), 1, None))
    assert "too many rows" in message(LIBRARY.hg_attention(C.byref(cache(pages=1 << 24, kv_heads=16)), C.byref(attention(heads=16)), 1, None))
    assert "dtype" in message(LIBRARY.hg_attention(C.byref(cache()), C.byref(attention()), 5, None))
    assert LIBRARY.hg_attention(C.byref(cache()), C.byref(attention(seqs=0)), 1, None) == 0


def test_a_workspace_is_asked_for_where_units_are_split_over_a_line():
    c = C.byref(cache(kv_heads=8, head_dim=128))
    assert LIBRARY.hg_attention_workspace(c, 0, 32, 100, 0) == 0 and LIBRARY.hg_attention_workspace(c, 1, 32, 500, 0) == 0
    assert LIBRARY.hg_attention_workspace(c, 512, 32, 16, 0) == 0                 # short sequences are not split
    size = LIBRARY.hg_attention_workspace(c, 512, 32, 64, 0)
    assert size > 0 and size % 16 == 0
    assert LIBRARY.hg_attention_workspace(c, 512, 32, 64, 16) == 0                # nor short windows
    assert LIBRARY.hg_attention_workspace(c, 4096, 32, 64, 0) == size             # as many slots as blocks


def test_python_calls_refuse_what_is_not_on_a_gpu():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    for call in (producer.norm_pack, producer.norm):
        with pytest.raises(ValueError, match="CUDA"):
            call(x, x[0])
    with pytest.raises(ValueError, match="CUDA"):
        PagedCache(torch.zeros(2, 1, page_bytes(16, 64), dtype=torch.uint8), 16, 64)
    with pytest.raises(ValueError, match="head_dim"):
        PagedCache(torch.zeros(2, 1, 100, dtype=torch.uint8), 16, 80)
    for bad in (dict(pages=0), dict(kv_heads=0), dict(page_size=0)):
        with pytest.raises(ValueError):
            PagedCache.allocate(**(dict(pages=2, page_size=16, kv_heads=1, head_dim=64, device="cpu") | bad))


class OnGpu(torch.Tensor):
    """Stands in for a tensor on a GPU where no kernel runs."""
    is_cuda = True


@pytest.mark.parametrize("scale, changes", [(1.0, False), (1 + 1e-9, False), (2 ** .5 * .5 ** .5, False), (1 + 2.0 ** -22, True), (0.0, True)])
def test_a_stream_is_returned_where_the_kernel_writes_one(scale, changes, monkeypatch):
    """The kernel decides by the scale in fp32."""
    calls = []

    class Library:
        @staticmethod
        def hg_norm(call, dtype, stream):
            calls.append(call._obj)
            return 0

    monkeypatch.setattr(native, "_host", None)
    monkeypatch.setattr(producer, "library", lambda: Library)
    monkeypatch.setattr(producer, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(producer, "_stream", lambda device: 0)
    x, weight = (torch.ones(shape, dtype=torch.bfloat16).as_subclass(OnGpu) for shape in ((2, 256), 256))
    for call in (producer.norm, producer.norm_pack):
        h = call(x, weight, scale=scale)[-1]
        assert (h is not x) == changes == (calls[-1].scale != 1.0) and bool(calls[-1].stream_out) == changes


class Layer:
    """Stands in for a layer and reads raw memory, so that a tensor without storage of its own is an error."""
    outputs, k = 3, 4

    def __call__(self, x):
        x.data_ptr()
        return x.detach().sum(1, keepdim=True).expand(-1, 3).contiguous()

    def linear(self, x, bias, activation, residual):
        y = self(x)
        for t in (bias, residual):
            if t is not None:
                t.data_ptr()
                y = y + t.detach()
        return y.relu() if activation == "relu" else y

    def takes_epilogue(self):
        return True


@pytest.fixture
def handle():
    number = ops.register_runtime(Layer())
    yield number
    ops._runtimes.pop(number)


X = torch.arange(8.).reshape(2, 4) - 4
BIAS, RESIDUAL = torch.tensor([1., 2., 3.]), torch.ones(2, 3)
WANT = (X.sum(1, keepdim=True) + BIAS + RESIDUAL).relu()


def test_the_registered_op(handle):
    call = lambda x, b, r: ops.linear_epilogue(x, handle, 3, b, "relu", r)  # noqa: E731
    assert torch.equal(call(X, BIAS, RESIDUAL), WANT)
    assert torch.equal(ops.linear_epilogue(X, handle, 3, None, "none", None), X.sum(1, keepdim=True).expand(-1, 3))
    for graph in (make_fx(call)(X, BIAS, RESIDUAL).graph, torch.fx.symbolic_trace(call).graph):
        names = [str(n.target) for n in graph.nodes if n.op == "call_function"]
        assert len(names) == 1 and names[0].startswith("hygemm_vllm.linear_epilogue"), names
    compiled = torch.compile(lambda x: call(x, BIAS, RESIDUAL) + 1, backend="aot_eager", fullgraph=True)
    assert torch.equal(compiled(X), WANT + 1)
    assert call(torch.empty(5, 4, device="meta"), BIAS.to("meta"), None).shape == (5, 3)
    for tensors in ((X.clone().requires_grad_(), BIAS, None), (X, BIAS.clone().requires_grad_(), None)):
        with pytest.raises(RuntimeError, match="no autograd formula"):
            call(*tensors).sum().backward()


def test_a_vllm_layers_bias(handle, monkeypatch):
    quantization = pytest.importorskip("hygemm_vllm.quantization")
    method = quantization.MixedLinearMethod(quantization.HyGEMMConfig.from_config({}), "m.q_proj")
    method.k, method.outputs, method.handle, method.runtime = 4, 3, handle, ops._runtimes[handle]
    bias = torch.nn.Parameter(BIAS)   # as vLLM makes it
    want = X.sum(1, keepdim=True) + BIAS
    calls = []
    original = Layer.linear
    monkeypatch.setattr(Layer, "linear", lambda self, *args: calls.append(args) or original(self, *args))
    for fuse in (False, True):
        monkeypatch.setattr(quantization, "FUSE_BIAS", fuse)
        with torch.inference_mode():
            assert torch.equal(method.apply(None, X, bias), want)
            assert torch.equal(method.apply(None, X.reshape(1, 2, 4), bias), want.reshape(1, 2, 3))
            assert torch.equal(method.apply(None, X), X.sum(1, keepdim=True).expand(-1, 3))
        assert len(calls) == 2 * fuse
        compiled = torch.compile(lambda x: method.apply(None, x, bias), backend="aot_eager", fullgraph=True)
        with torch.inference_mode():
            assert torch.equal(compiled(X), want)
        torch._dynamo.reset()
        calls.clear()
    strided = torch.stack([BIAS, BIAS], 1)[:, 0]   # what the epilogue does not take is added behind the layer as ever
    assert torch.equal(method.apply(None, X, bias.double()), want.double()) and torch.equal(method.apply(None, X, strided), want) and not calls
    monkeypatch.setattr(Layer, "takes_epilogue", lambda self: False)
    assert torch.equal(method.apply(None, X, bias), want) and not calls


def test_what_asks_for_a_gradient():
    """Recorded gradients and tangents of forward mode; neither where it is off."""
    x, tangent = torch.randn(2, 4), torch.ones(2, 4)
    assert not native._differentiated(x, None) and not native._differentiated()
    leaf = x.clone().requires_grad_()
    assert native._differentiated(None, leaf)
    with torch.no_grad():
        assert not native._differentiated(leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, tangent)
        assert native._differentiated(x, dual) and not native._differentiated(x)
        with torch.no_grad():
            assert native._differentiated(dual)      # turns recording off, tangents not
        with torch.inference_mode():
            assert not native._differentiated(dual)
        with forward_ad._set_fwd_grad_enabled(False):
            assert not native._differentiated(dual)
    assert not native._differentiated(dual)
    seen = []
    torch.func.jvp(lambda t: seen.append(native._differentiated(t)) or t.sum(), (x,), (tangent,))
    assert seen == [True]


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
def test_tensors_without_memory_are_refused():
    """As tracing has them: their address is zero, which would stand for an operand that is not there."""
    with FakeTensorMode():
        x, weight = torch.empty(2, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(256, dtype=torch.bfloat16, device="cuda")
        held = PagedCache(torch.empty(4, 2, page_bytes(16, 64), dtype=torch.uint8, device="cuda"), 16, 64)
        kv, slots = torch.empty(2, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(2, dtype=torch.int64, device="cuda")
        table, lengths = torch.empty(2, 3, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    for call in (lambda: producer.norm(x, weight), lambda: producer.norm_pack(x, weight, residual=x), lambda: held.write(kv, kv, slots),
                 lambda: held.read(slots), lambda: held.attention(kv, table, lengths), lambda: held.attention_pack(kv, table, lengths)):
        with pytest.raises(ValueError, match="in memory"):
            call()


@pytest.mark.parametrize("missing", ["residual", "gate", "post_weight", "weight"])
def test_an_operand_without_memory_is_not_left_out(missing):
    class Nowhere(OnGpu):
        def data_ptr(self):
            return 0

    operands = {name: torch.ones(shape, dtype=torch.bfloat16).as_subclass(Nowhere if name == missing else OnGpu)
                for name, shape in (("x", (2, 256)), ("weight", 256), ("residual", (2, 256)), ("gate", 256), ("post_weight", 256))}
    with pytest.raises(ValueError, match="in memory"):
        producer._norm(operands["x"], operands["weight"], 1e-6, operands["residual"], operands["gate"], 1.0, operands["post_weight"], None, True)
