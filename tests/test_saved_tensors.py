"""Backward passes under saved-tensor hooks, which may return other strides and
addresses than the forward pass saved.

On the CPU the library's calls are recorded: what a backward pass hands to the
library has to describe the tensors that came back (a view's strides against
its tensor's, then its values).  On the GPU gradients under hooks equal those
without, bit for bit: the same kernels read the same values."""
import contextlib
import ctypes

import pytest
import torch

from gpu_util import DEV

gpu = pytest.mark.gpu
INT = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}


def bits(x):
    return x.contiguous().view(INT[x.element_size()])


def memory(address, shape, strides, dtype):
    """The tensor at an address of this process."""
    size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    raw = (ctypes.c_char * (size * dtype.itemsize)).from_address(address)
    return torch.as_strided(torch.frombuffer(raw, dtype=dtype), shape, strides).clone()


class Recorder:
    """Stands in for the library: runs nothing, checks what a backward pass is given."""

    def __init__(self, real):
        self.real = real
        self.returned = {}  # by address: the tensors that hooks returned
        self.expected = None  # the values that the forward pass saved, by name
        self.checked = 0

    def __getattr__(self, name):
        if name.endswith("_bytes") or name == "b2_last_error":
            return getattr(self.real, name)
        if name.endswith("_backward"):
            return lambda *args: self.backward(name, args)
        return lambda *args: 0

    def backward(self, name, args):
        from b200_pisa import _lib

        views = {"b2_attention_backward": ("q", "k", "v", "out", "low", "dout"),
                 "b2_qk_norm_rope_backward": ("q", "k", "dout", "dout2"),
                 "b2_norm_rope_attention_backward": ("q", "k", "v", "out", "low", "dout")}[name]
        for key, packed in zip(views, args):
            if packed is None:
                continue
            view = _lib.View.from_buffer_copy(packed)
            shape = (view.batch, view.heads, view.tokens, view.head_dim)
            strides = (view.stride_b, view.stride_h, view.stride_t, 1)
            self.compare(key, view.base, shape, strides)
        flat = {"b2_attention_backward": {"lse": 6, "lens": 12},
                "b2_qk_norm_rope_backward": {"wq": 6, "wk": 7},
                "b2_norm_rope_attention_backward": {"lse": 6, "wq": 7, "wk": 8, "lens": 14, "saved": 15}}[name]
        for key, i in flat.items():
            if args[i] is not None:
                shape = self.expected[key].shape
                self.compare(key, args[i], shape, torch.empty(shape, device="meta").stride())
        rotary = {"b2_qk_norm_rope_backward": 10, "b2_norm_rope_attention_backward": 11}.get(name)
        if rotary is not None:
            r = _lib.Rotary.from_buffer_copy(args[rotary])
            batch, (tokens, axes) = self.expected["q"].shape[0], self.expected["pos"].shape[-2:]
            self.compare("pos", r.positions, (batch, tokens, axes), (r.stride_b, r.stride_t, r.stride_axis))
        return 0

    def compare(self, key, address, shape, strides):
        if key in ("dout", "dout2"):
            return
        tensor = self.returned.get(address)
        if tensor is not None:  # before its memory is read by these strides
            inside = sum((n - 1) * s for n, s in zip(shape, strides)) * tensor.element_size()
            assert address + inside < tensor.untyped_storage().data_ptr() + tensor.untyped_storage().nbytes(), key
            given = [s for n, s in zip(shape, strides) if n > 1 and s != 0]
            assert given == [s for n, s in zip(tensor.shape, tensor.stride()) if n > 1 and s != 0], (key, strides, tensor.stride())
        want = self.expected[key]
        assert torch.equal(bits(memory(address, shape, strides, want.dtype)), bits(want.expand(shape))), key
        self.checked += 1


def contiguous(x):
    return x.clone(memory_format=torch.contiguous_format)


def unaligned(x):
    """Contiguous, from an address off the 16-byte boundaries."""
    flat = torch.empty(x.numel() + 64, dtype=x.dtype, device=x.device)
    start = next(i for i in range(64) if (flat.data_ptr() + i * x.element_size()) % 16 == (8 if x.element_size() > 4 else 4))
    return flat[start:start + x.numel()].view(x.shape).copy_(x)


def turned(x):
    """The dimensions' order in memory reversed."""
    return x.permute(*reversed(range(x.ndim))).contiguous().permute(*reversed(range(x.ndim)))


HOOKS = {"contiguous": contiguous, "unaligned": unaligned, "turned": turned, "padded": lambda x: torch.nn.functional.pad(
    x, (0, 8) if x.ndim == 4 else (0, 0))[..., :x.shape[-1]]}


def inputs(dev, batch=2, heads=4, kv_heads=4, tokens=70, dim=64):
    gen = torch.Generator(device=dev).manual_seed(5)
    fused = torch.randn(batch, tokens, 3, heads, dim, generator=gen, device=dev).to(torch.bfloat16)
    q, k, v = (fused[:, :, i, :n].permute(0, 2, 1, 3) for i, n in enumerate((heads, kv_heads, kv_heads)))
    wq, wk = (1 + 0.1 * torch.randn(dim, generator=gen, device=dev).to(torch.bfloat16) for _ in range(2))
    pos = torch.stack([torch.arange(tokens, device=dev) // n for n in (7, 1)], 1)[None].expand(batch, -1, -1)
    lens = torch.tensor([tokens, 9][:batch], dtype=torch.int32, device=dev)
    return [x.detach().requires_grad_() for x in (q, k, v, wq, wk)] + [pos, lens]


def run(op, q, k, v, wq, wk, pos, lens):
    import b200_pisa

    if op == "qk_norm_rope":
        return b200_pisa.qk_norm_rope(q, k, wq, wk, pos, (32, 32), interleaved=False), (q, k, wq, wk)
    if op == "axial_rope":
        return (b200_pisa.axial_rope(q, pos, (32, 16)),), (q,)
    if op == "attention":
        return (b200_pisa.attention(q, k, v, causal=True, key_lengths=lens),), (q, k, v)
    if op == "flat attention":
        return (b200_pisa.attention(q[:, 0], k[:, 1], v[:, 2], 0.3),), (q, k, v)
    return (b200_pisa.norm_rope_attention(q, k, v, wq, wk, pos, (32, 32), key_lengths=lens),), (q, k, v, wq, wk)


@pytest.fixture
def recorded(monkeypatch):
    import b200_pisa
    from b200_pisa import exact, fused, rotary

    recorder = Recorder(b200_pisa.LIB)
    for module in (exact, fused, rotary):
        monkeypatch.setattr(module, "LIB", recorder)
        monkeypatch.setattr(module, "on_device", lambda x: contextlib.nullcontext())
        monkeypatch.setattr(module, "raw_stream", lambda x: 0)
        monkeypatch.setattr(module, "require_one_device", lambda *args: None)
    return recorder


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("op", ["attention", "flat attention", "qk_norm_rope", "norm_rope_attention"])
def test_the_library_is_given_what_came_back(recorded, op, hook):
    tensors = inputs("cpu")
    packed = []

    def pack(x):
        packed.append(x.detach().clone())
        return x

    def unpack(x):
        got = HOOKS[hook](x)
        recorded.returned[got.data_ptr()] = got
        return got

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        outs, leaves = run(op, *tensors)
    # the order that each operator saves them in
    names = {"qk_norm_rope": ("q", "k", "wq", "wk", "pos"),
             "norm_rope_attention": ("q", "k", "v", "wq", "wk", "pos", "out", "lse", "low", "saved", "lens"),
             "attention": ("q", "k", "v", "out", "lse", "low", "lens"),
             "flat attention": ("q", "k", "v", "out", "lse")}[op]
    assert len(packed) == len(names)
    recorded.expected = dict(zip(names, packed))
    torch.autograd.backward(outs, [torch.ones_like(x) for x in outs])
    assert recorded.checked == len(packed)
    assert all(x.grad.shape == x.shape for x in leaves)


@pytest.mark.parametrize("op", ["attention", "qk_norm_rope", "norm_rope_attention"])
@pytest.mark.parametrize("change", [lambda x: x[..., :-8] if x.shape[-1] == 64 else x,
                                    lambda x: x.float() if x.dtype == torch.bfloat16 else x], ids=["shape", "dtype"])
def test_other_shapes_and_types_are_refused(recorded, op, change):
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, change):
        outs, _ = run(op, *inputs("cpu"))
    with pytest.raises(ValueError, match="another shape or dtype"):
        torch.autograd.backward(outs, [torch.ones_like(x) for x in outs])


@pytest.mark.parametrize("op", ["attention", "qk_norm_rope", "norm_rope_attention"])
def test_another_device_is_refused(recorded, monkeypatch, op):
    from b200_pisa import _args, exact, fused, rotary

    outs, _ = run(op, *inputs("cpu"))
    for module in (exact, fused, rotary):
        monkeypatch.setattr(module, "require_one_device", _args.require_one_device)
    with pytest.raises(ValueError, match="one CUDA device"):  # nothing here is on one
        torch.autograd.backward(outs, [torch.ones_like(x) for x in outs])


@gpu
@pytest.mark.parametrize("hook", [*HOOKS, "save_on_cpu", "save_on_cpu pinned"])
@pytest.mark.parametrize("op", ["axial_rope", "qk_norm_rope", "attention", "flat attention", "norm_rope_attention"])
def test_gradients_under_hooks(op, hook):
    from b200_pisa import _lib

    tensors = inputs(DEV)
    outs, leaves = run(op, *tensors)
    douts = [torch.randn_like(x) for x in outs]
    want = torch.autograd.grad(outs, leaves, douts)
    hooks = (torch.autograd.graph.save_on_cpu(pin_memory=hook.endswith("pinned")) if hook.startswith("save_on_cpu")
             else torch.autograd.graph.saved_tensors_hooks(lambda x: x, HOOKS[hook]))
    with hooks:
        outs, leaves = run(op, *tensors)
    got = torch.autograd.grad(outs, leaves, douts)
    assert all(torch.equal(a, b) and a.stride() == b.stride() for a, b in zip(got, want))
    _lib.check_status()


@gpu
@pytest.mark.parametrize("op", ["axial_rope", "qk_norm_rope", "attention", "flat attention", "norm_rope_attention"])
def test_gradients_under_checkpointing(op):
    """The forward pass runs again and hands over its own saved tensors."""
    from torch.utils.checkpoint import checkpoint

    *leaves, pos, lens = inputs(DEV)
    outs, used = run(op, *leaves, pos, lens)
    douts = [torch.randn_like(x) for x in outs]
    want = torch.autograd.grad(outs, used, douts)
    outs = checkpoint(lambda *x: run(op, *x, pos, lens)[0], *leaves, use_reentrant=False)
    got = torch.autograd.grad(outs, used, douts)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("how", ["no leaf wants one", "no_grad"])
@pytest.mark.parametrize("op", ["axial_rope", "qk_norm_rope", "attention", "flat attention", "norm_rope_attention"])
def test_calls_without_gradients_keep_their_results_alone(op, how):
    tensors = inputs(DEV, tokens=700)
    if how != "no_grad":
        tensors = [x.detach() for x in tensors]
    with torch.no_grad() if how == "no_grad" else contextlib.nullcontext():
        run(op, *tensors)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(DEV)
        outs, _ = run(op, *tensors)
        torch.cuda.synchronize()
    kept = torch.cuda.memory_allocated(DEV) - before
    rounded = sum(-(-x.numel() * x.element_size() // 512) * 512 for x in outs)
    assert kept == rounded and not any(x.requires_grad for x in outs)
