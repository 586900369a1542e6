"""AdamW over many tensors at once and the norm of their gradients, on libnerfhip.so (nerfhip_adamw_*, include/nerfhip.h).

Tensors are torch device tensors, used as owners of device memory.  Calls follow torch's current stream of the tensors'
device unless set_stream names another; nothing synchronises, so a step may be captured into a graph (its update count and,
where given, its learning rate and gradient factor live on the device)."""
import ctypes as C
import itertools
import math

from . import _lib

BLOCK = 256     # values that share a scale of an 8-bit state


def _dtype_code(t):
    import torch
    return {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}.get(t)


def _current_stream(device):
    """Address of torch's current stream; 0: HIP's default stream."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # a tenth of the time of building a Stream object
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


class _Handle:
    """A C handle of kind `_kind` ("adamw", "ffn"): errors, streams, lifetime."""
    _kind = ""

    def __init__(self, device):
        self._lib = _lib.load()
        self._h = None
        self.device = int(device)
        self._stream = None      # what the handle was last told
        self._fixed = None       # the stream that set_stream named

    def _fn(self, name):
        return getattr(self._lib, f"nerfhip_{self._kind}_{name}")

    def _chk(self, rc, what):
        if rc != 0:
            msg = self._fn("last_error")(self._h)
            raise _lib.NerfHipError(f"{self._kind} {what} failed (code {rc}): {msg.decode() if msg else '?'}")

    def close(self):
        if getattr(self, "_h", None):
            self._fn("destroy")(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_stream(self, stream_ptr):
        """Run on this HIP stream from now on; None: on torch's current stream again.  New tensors (results, scratch memory) then belong
        to that stream.  It has to exist until a call has run on another one: what synchronises waits for the last call's stream."""
        import torch
        self._fixed = None if stream_ptr is None else torch.cuda.ExternalStream(stream_ptr, device=self._device)
        if stream_ptr is not None:
            self._stream = stream_ptr or _lib.STREAM_DEFAULT
            self._chk(self._fn("set_stream")(self._h, self._stream), "set_stream")

    def synchronize(self):
        self._chk(self._fn("synchronize")(self._h), "synchronize")

    def _follow(self):
        """Without set_stream: torch's current stream of the handle's device."""
        if self._fixed is not None:
            return
        s = _current_stream(self.device) or _lib.STREAM_DEFAULT
        if s != self._stream:
            self._chk(self._fn("set_stream")(self._h, s), "set_stream")
            self._stream = s

    def _empty(self, shape, dtype):
        """A tensor of the stream that the handle runs on: torch hands its memory out again only in that stream's order."""
        import torch
        if self._fixed is None:
            return torch.empty(shape, dtype=dtype, device=self._device)
        with torch.cuda.stream(self._fixed):
            return torch.empty(shape, dtype=dtype, device=self._device)

    def _on_device(self, t, name):
        if t.device.type != "cuda" or t.device.index != self.device:
            raise ValueError(f"{name}: expected a tensor on cuda:{self.device}, got {t.device}")


class AdamW(_Handle):
    """AdamW(params, grads): one launch updates all of them.

    params, grads   contiguous tensors of the same sizes; all params of one type (float32, bfloat16, float16), all grads of
                    that type or float32.  The object keeps their addresses: write gradients into the same tensors.
    weight_decay    one number, or one for each tensor
    state_bits      32, or 8: first moments as float8_e4m3fn and roots of second moments as uint8 codes, with a float32 scale
                    for each 256 values (include/nerfhip.h has the codes)
    master          float32 copies of 16-bit params, which the step updates and rounds into them
    state           tensors to use instead of new ones: {"exp_avg", "exp_avg_sq"[, "exp_avg_scale", "exp_avg_sq_scale"]
                    [, "master"]}, a list for each"""
    _kind = "adamw"

    def __init__(self, params, grads, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, master=False,
                 state=None, step=0):
        import torch
        self.params, self.grads = list(params), list(grads)
        if not self.params or len(self.params) != len(self.grads):
            raise ValueError("params and grads must be lists of the same length, one tensor at least")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        super().__init__(self.params[0].device.index if self.params[0].device.type == "cuda" else 0)
        n = len(self.params)
        pt, gt = self.params[0].dtype, self.grads[0].dtype
        if _dtype_code(pt) is None or gt not in (pt, torch.float32):
            raise ValueError(f"unsupported types: params {pt}, grads {gt}")
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        if len(decay) != n:
            raise ValueError("weight_decay must be one number or one for each tensor")
        self.lr, self.state_bits, self.master = float(lr), state_bits, bool(master)
        sizes = [p.numel() for p in self.params]
        blocks = [-(-k // BLOCK) for k in sizes]
        self.state_offsets = list(itertools.accumulate([0] + [BLOCK * b for b in blocks[:-1]]))
        self.state_size = BLOCK * sum(blocks)
        want = {"exp_avg": (torch.float8_e4m3fn if state_bits == 8 else torch.float32, sizes),
                "exp_avg_sq": (torch.uint8 if state_bits == 8 else torch.float32, sizes)}
        if state_bits == 8:
            want.update(exp_avg_scale=(torch.float32, blocks), exp_avg_sq_scale=(torch.float32, blocks))
        if self.master:
            want["master"] = (torch.float32, sizes)
        if state is None:
            for i, (p, g) in enumerate(zip(self.params, self.grads)):
                self._on_device(p, f"params[{i}]")
            new = lambda t, k: torch.zeros(k, dtype=torch.uint8, device=f"cuda:{self.device}").view(t) if t.itemsize == 1 else \
                torch.zeros(k, dtype=t, device=f"cuda:{self.device}")  # noqa: E731
            state = {k: [new(t, m) for m in ms] for k, (t, ms) in want.items()}
            if self.master:
                state["master"] = [p.detach().float().reshape(-1).contiguous() for p in self.params]
        if set(state) != set(want):
            raise ValueError(f"state must have {sorted(want)}, got {sorted(state)}")
        self.state = {k: list(state[k]) for k in want}
        groups = {"params": (self.params, pt, sizes), "grads": (self.grads, gt, sizes)}
        groups.update({k: (self.state[k], t, m) for k, (t, m) in want.items()})
        for name, (tensors, t, ms) in groups.items():
            if len(tensors) != n:
                raise ValueError(f"{name}: expected {n} tensors, got {len(tensors)}")
            for i, (x, m) in enumerate(zip(tensors, ms)):
                self._on_device(x, f"{name}[{i}]")
                if x.dtype != t or x.numel() != m or not x.is_contiguous():
                    raise ValueError(f"{name}[{i}]: expected {m} contiguous values of {t}, got {x.numel()} of {x.dtype}")
        table = (_lib.AdamWTensor * n)()
        for i in range(n):
            e = table[i]
            e.param, e.grad, e.n, e.weight_decay = self.params[i].data_ptr(), self.grads[i].data_ptr(), sizes[i], float(decay[i])
            e.m, e.v = self.state["exp_avg"][i].data_ptr(), self.state["exp_avg_sq"][i].data_ptr()
            if state_bits == 8:
                e.m_scale, e.v_scale = self.state["exp_avg_scale"][i].data_ptr(), self.state["exp_avg_sq_scale"][i].data_ptr()
            if self.master:
                e.master = self.state["master"][i].data_ptr()
        cfg = _lib.AdamWConfig(betas[0], betas[1], eps, _dtype_code(pt), _dtype_code(gt), state_bits, int(self.master), self.device)
        h = C.c_void_p()
        self._chk(self._fn("create")(C.byref(cfg), table, n, C.byref(h)), "create")
        self._h = h
        self._device = torch.device("cuda", self.device)
        if step:
            self.set_step(step)

    def _scalar(self, t, name):
        import torch
        self._on_device(t, name)
        if t.dtype != torch.float32 or t.numel() < 1 or not t.is_contiguous():
            raise ValueError(f"{name}: expected a float32 tensor of one value")
        return t.data_ptr()

    def step(self, lr=None, grad_scale=None):
        """One update.  lr: a number, or a float32 device tensor that is read when the kernel runs.  grad_scale: a float32 device
        tensor, a factor on every gradient; if it is not finite nothing is changed or counted."""
        self._follow()
        lr = self.lr if lr is None else lr
        lr_dev = self._scalar(lr, "lr") if hasattr(lr, "data_ptr") else None
        if lr_dev is None and not math.isfinite(lr):
            raise ValueError("lr must be finite")
        gs = None if grad_scale is None else self._scalar(grad_scale, "grad_scale")
        self._chk(self._fn("step")(self._h, 0.0 if lr_dev else float(lr), lr_dev, gs), "step")

    def grad_norm(self, max_norm=None, loss_scale=1.0, out=None):
        """float32 tensor [norm, factor]: the norm of all gradients divided by loss_scale, and what step() takes as grad_scale
        (norm[1:]) to undo the loss scale and to clip to max_norm; NaN if the norm is not finite."""
        import torch
        self._follow()
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be > 0")
        if out is None:
            out = self._empty(2, torch.float32)
        elif out.numel() < 2:
            raise ValueError("out: expected two values")
        self._chk(self._fn("grad_norm")(self._h, float(max_norm or 0.0), float(loss_scale), self._scalar(out, "out")), "grad_norm")
        return out

    def read_state(self, moments=True, roots=True):
        """(m, sqrt(v)) of all tensors as numbers: two flat float32 tensors (None where not asked for) in which tensor i starts at
        state_offsets[i], a multiple of 256; zeros in between.  For checkpoints that other programs read."""
        import torch
        self._follow()
        new = lambda want: self._empty(self.state_size, torch.float32) if want else None  # noqa: E731
        m, r = new(moments), new(roots)
        self._chk(self._fn("read_state")(self._h, m.data_ptr() if moments else None, r.data_ptr() if roots else None), "read_state")
        return m, r

    def _wait(self):
        """For calls that synchronise: whatever stream the last call ran on has to be done with, not just the current one."""
        self.synchronize()
        self._follow()

    def get_step(self):
        """The number of updates so far.  Waits for the last call's stream and the current one; a graph that is replayed on a third has to
        be waited for before."""
        self._wait()
        t = C.c_int64()
        self._chk(self._fn("get_step")(self._h, C.byref(t)), "get_step")
        return t.value

    def set_step(self, step):
        """Makes this the number of updates so far; waits as get_step does."""
        self._wait()
        self._chk(self._fn("set_step")(self._h, int(step)), "set_step")

    def state_dict(self):
        """The state's tensors (not copies) and the update count: what a checkpoint holds."""
        return {"step": self.get_step(), "state_bits": self.state_bits, **{k: list(v) for k, v in self.state.items()}}

    def load_state_dict(self, d):
        """Copies a state_dict's values into this object's tensors; waits for the steps before and for the copies."""
        import torch
        if d["state_bits"] != self.state_bits or any(len(d.get(k, ())) != len(v) for k, v in self.state.items()):
            raise ValueError("the state_dict is of other tensors or of another state_bits")
        for k, v in self.state.items():
            for i, (x, y) in enumerate(zip(v, d[k])):
                if x.dtype != y.dtype or x.numel() != y.numel():
                    raise ValueError(f"{k}[{i}]: expected {x.numel()} values of {x.dtype}, got {y.numel()} of {y.dtype}")
        self.synchronize()
        for k, v in self.state.items():
            for x, y in zip(v, d[k]):
                x.copy_(y.reshape(x.shape))
        torch.cuda.current_stream(self._device).synchronize()      # set_stream may have named another for the steps
        self.set_step(d["step"])
