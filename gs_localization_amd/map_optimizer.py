"""The optimiser step of a Gaussian map and the pruning that goes with it, on hand-written HIP kernels (include/gsr.h: gsr_grad_norm,
gsr_adamw_step, gsr_adamw_moments, gsr_evict_rows).

gaussian_splatting/train.py:155-157 steps torch.optim.Adam over the six tensors of a map and gaussian_splatting/scene/
gaussian_model.py:269-328 rewrites its state whenever splats are pruned or added.  Here

  AdamW           an optimiser with torch's constructor, groups and state ("exp_avg", "exp_avg_sq"): one launch for all tensors; moments
                  in 32 bits or in a byte each (state_bits=8: 16 instead of 28 bytes of traffic per fp32 parameter, 2 instead
                  of 8 bytes of state); clipping by the gradients' norm without a read-back; evict() and append_rows() for its maps
  grad_norm, adamw_step, adamw_step_8bit, moments_8bit, evict_rows      the operators by themselves
  compositing_weights                                                   what evict_rows accumulates, from the rasterizer

No operator reads anything back, and each runs on its tensors' device and that device's current stream; two steps of the same tensors
must not overlap, as with any operation in place.  (compositing_weights is a forward and a backward of the rasterizer, which may read back and is not made
for capture.)  Nothing falls back to torch or to the CPU: tensors elsewhere are refused.  Tensors that a step writes must be contiguous and must not overlap (refused); the
step counts live on the device, so a captured graph counts on when it is replayed."""
import ctypes as C
import math
import struct

import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_OPT = struct.Struct("7Q2dq2i")          # gsr_opt_tensor
_ORIGIN = struct.Struct("2dI4x")         # gsr_code_origin
_MOMENT = struct.Struct("5Qq")           # gsr_moment_tensor
_ROW = struct.Struct("4Qq")              # gsr_row_tensor
WINDOW = 256                             # elements that share a window byte of the 8-bit root


def _no_device(tensors, name):
    """Says why the tensors are not all on one HIP device."""
    dev = None
    for t in tensors:
        if not torch.is_tensor(t):
            raise TypeError(f"{name} needs tensors, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"{name} needs HIP tensors (there is no CPU path)")
        if dev is not None and t.device != dev:
            raise RuntimeError(f"{name}: tensors on {dev} and {t.device}")
        dev = t.device


def _device(tensors, name):
    """The number of the one HIP device that all of them live on."""
    try:
        index = tensors[0].get_device()
        if index >= 0 and all([t.get_device() == index for t in tensors]):
            return index
    except AttributeError:
        pass
    _no_device(tensors, name)
    raise RuntimeError(f"{name}: no device")


def _type(t, name):
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{name}: {t.dtype} is not supported (float32, bfloat16, float16)") from None


class _on:
    """Device `index` as the current one; gives its current stream."""

    def __init__(self, index):
        self.index = index
        self.back = torch.cuda.current_device()

    def __enter__(self):
        if self.index != self.back:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.index != self.back:
            torch.cuda.set_device(self.back)


# (the handle without a torch.cuda.Stream around it: 0.2 us for 3.5, in calls of some 20)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _workspace(nbytes, index):
    t = torch.empty(nbytes, dtype=torch.uint8, device=f"cuda:{index}")
    return t, _lib.FixedBuffer(t.data_ptr(), nbytes, 0)


def _dense(t):
    """t, or a dense copy of its values: of strides, and of what torch has only marked (a conjugate; the sign of its imaginary part, which is
    contiguous only as one element)."""
    if t.is_contiguous() and not t.is_neg() and not t.is_conj():
        return t
    return t.resolve_conj().resolve_neg().contiguous()


def _address(buf):
    return C.addressof(C.c_char.from_buffer(buf)) if buf else None


def grad_norm(grads, max_norm=math.inf):
    """grads: tensors (float32, bfloat16, float16; any sizes).  Returns a float32 tensor (norm, coefficient) on their device: the 2-norm over
    all of them (64-bit sums in a fixed order) and min(1, max_norm / (norm + 1e-6)), what torch.nn.utils.clip_grad_norm_ would multiply them
    by -- handed to adamw_step as `clip` no gradient is written.  A NaN or infinite gradient gives a norm that says so."""
    lib = _lib.load()
    grads = [g if g.is_contiguous() and not g.is_neg() else _dense(g) for g in grads]
    if not grads:
        raise ValueError("grad_norm: no gradients")
    if not max_norm >= 0.0:
        raise ValueError(f"grad_norm: max_norm >= 0 required, got {max_norm}")
    index = _device(grads, "grad_norm")
    n = len(grads)
    types = (C.c_int * n)(*[_type(g, "grad_norm") for g in grads])
    ptrs = (C.c_void_p * n)(*[g.data_ptr() for g in grads])
    numels = (C.c_longlong * n)(*[g.numel() for g in grads])
    with _on(index) as stream:
        out = torch.empty(2, dtype=torch.float32, device=grads[0].device)
        keep, ws = _workspace(lib.gsr_grad_norm_bytes(n), index)
        _lib.check(lib.gsr_grad_norm(n, ptrs, numels, types, max_norm, out.data_ptr(), _lib.fixed_buffer_fn(), C.addressof(ws), stream))
    return out


def _per_tensor(x, n, name):
    if isinstance(x, (list, tuple)):
        if len(x) != n:
            raise ValueError(f"{name}: {len(x)} values for {n} tensors")
        return x
    return [x] * n


def _pack(bits, name, params, grads, state0, state1, windows, clocks, lr, betas, eps, weight_decay, clip, seed, origin=None):
    """A call of gsr_adamw_step_coded for _launch, its tensors checked; None without tensors."""
    n = len(params)
    if not (len(grads) == len(state0) == len(state1) == len(clocks) == n) or (windows is not None and len(windows) != n):
        raise ValueError(f"{name}: lists of different lengths")
    if n == 0:
        return None
    lrs, decays = _per_tensor(lr, n, name + ": lr"), _per_tensor(weight_decay, n, name + ": weight_decay")
    d0, d1 = (torch.float32, torch.float32) if bits == 32 else (torch.uint8, torch.int8)
    index = _device(params, name)
    if clip is not None and not (clip.dtype is torch.float32 and clip.numel() == 2 and clip.is_contiguous() and clip.get_device() == index):
        raise ValueError(f"{name}: clip is grad_norm's result (two float32 on the parameters' device)")
    buf, keep, origins = bytearray(_OPT.size * n), [], None
    if origin is not None:          # (8 bits) a tensor's: the betas it was stored with, its place
        origins = bytearray(_ORIGIN.size * n)
        for i, ((b1, b2), place) in enumerate(origin):
            _ORIGIN.pack_into(origins, _ORIGIN.size * i, b1, b2, place)
    for i in range(n):
        p, g, a, b, clock, rate = params[i], grads[i], state0[i], state1[i], clocks[i], lrs[i]
        w = None if windows is None else windows[i]
        k = p.numel()
        if not (g.get_device() == a.get_device() == b.get_device() == clock.get_device() == index and (w is None or w.get_device() == index)):
            _no_device((p, g, a, b, clock) if w is None else (p, g, a, b, clock, w), name)
        if a.dtype is not d0 or b.dtype is not d1 or clock.dtype is not torch.float64 or (w is not None and w.dtype is not torch.uint8):
            raise TypeError(f"{name}: tensor {i}: moments are {d0} and {d1}, the clock float64" + (", the window uint8" if bits == 8 else ""))
        if g.shape != p.shape or a.numel() != k or b.numel() != k or clock.numel() != 4 or (w is not None and w.numel() != (k + WINDOW - 1) // WINDOW):
            raise ValueError(f"{name}: tensor {i}: sizes do not match the parameter's {tuple(p.shape)}")
        if not (p.is_contiguous() and a.is_contiguous() and b.is_contiguous() and clock.is_contiguous() and (w is None or w.is_contiguous())):
            raise ValueError(f"{name}: tensor {i}: what the step writes must be contiguous")
        if k == 1 and p.is_neg():
            raise ValueError(f"{name}: tensor {i}: the parameter is marked as a negative: resolve_neg() first")
        if not g.is_contiguous() or (k == 1 and g.is_neg()):
            g = _dense(g)
            keep.append(g)
        pt, gt = _TYPES.get(p.dtype), _TYPES.get(g.dtype)
        if pt is None or gt is None:
            _type(p, name), _type(g, name)
        lr_ptr = 0
        if not isinstance(rate, float) and torch.is_tensor(rate):
            if not (rate.dtype is torch.float64 and rate.numel() == 1 and rate.get_device() == index):
                raise ValueError(f"{name}: lr as a tensor is one float64 on the parameters' device")
            lr_ptr, rate = rate.data_ptr(), 0.0
        _OPT.pack_into(buf, _OPT.size * i, p.data_ptr(), g.data_ptr(), a.data_ptr(), b.data_ptr(), 0 if w is None else w.data_ptr(),
                       clock.data_ptr(), lr_ptr, rate, decays[i], k, pt, gt)
    args = _lib.AdamwArgs(n, bits, _address(buf), betas[0], betas[1], eps, None if clip is None else clip.data_ptr(), seed & 0xFFFFFFFF, None)
    # (the last: what has to stay alive until the launch)
    return args, origins, index, [*params, *state0, *state1, *clocks, *(windows or ())], (buf, keep, clip)


def _launch(call):
    args, origins, index, written, _ = call
    with _on(index) as stream:
        args.stream = stream
        _lib.check(_lib.load().gsr_adamw_step_coded(C.byref(args), _address(origins)))
    torch.autograd.graph.increment_version(written)


def _step(*args):
    call = _pack(*args)
    if call is not None:
        _launch(call)


def new_clock(device):
    """The step count of one tensor: beta1^t, beta2^t, t and a word of the kernel's own, in 64 bits on the device."""
    return torch.tensor([1.0, 1.0, 0.0, 0.0], dtype=torch.float64, device=device)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, clocks, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, clip=None):
    """One AdamW step over many tensors in one launch, in place (torch.optim.AdamW; with weight_decay 0 torch.optim.Adam).
    params, grads: float32, bfloat16 or float16; exp_avgs, exp_avg_sqs: float32, zero before the first step; clocks: new_clock() each.
    lr, weight_decay: one number or one per tensor; an lr may be a float64 tensor of one element on the device, which a replayed graph
    reads anew.  clip: what grad_norm returned, or None.  A gradient that is not contiguous is copied.
    A clock holds the products of its steps' betas; torch's corrections are 1 - beta ** t of the current ones, which differs only where
    betas change between steps: set clock[0] and clock[1] anew then (AdamW does)."""
    _step(32, "adamw_step", params, grads, exp_avgs, exp_avg_sqs, None, clocks, lr, betas, eps, weight_decay, clip, 0)


def adamw_step_8bit(params, grads, rms, ratio, window, clocks, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, clip=None, seed=0, state_betas=None):
    """adamw_step with a byte for each moment: rms (uint8, sqrt(exp_avg_sq) to a sixteenth of its binade), ratio (int8, exp_avg / sqrt(exp_avg_sq)
    in 127 steps of the largest it can be), window (uint8, one per 256 elements of the flattened tensor: which sixteen binades rms
    covers); all zero before the first step.  Rounding is stochastic, from `seed`, the step, the tensor's place in the list and the element's: the same
    call on the same state gives the same bits.  Needs beta1^2 < beta2.  moments_8bit reads them.
    With beta2 = 0.999 the stored root walks about the 32-bit moment's with a standard deviation of a tenth, and so does each element's rate.
    The largest that the ratio can be depends on the betas.  state_betas: those of the last step that stored the ratios, one pair or one per
    tensor, where they are not this step's; ratios are read with them and stored with `betas`."""
    if state_betas is not None:
        state_betas = _per_tensor(state_betas if isinstance(state_betas[0], (list, tuple)) else [state_betas] * len(params), len(params), "adamw_step_8bit: state_betas")
    _step(8, "adamw_step_8bit", params, grads, rms, ratio, window, clocks, lr, betas, eps, weight_decay, clip, seed,
          None if state_betas is None else zip(state_betas, range(len(params))))


def moments_8bit(rms, ratio, window, betas=(0.9, 0.999), dtype=torch.float32):
    """The moments that adamw_step_8bit's bytes stand for, as two lists of tensors: exp_avg and sqrt(exp_avg_sq).  betas: those of the step that
    stored them."""
    lib = _lib.load()
    n = len(rms)
    if len(ratio) != n or len(window) != n:
        raise ValueError("moments_8bit: lists of different lengths")
    if dtype not in _TYPES:
        raise TypeError(f"moments_8bit: {dtype} is not supported (float32, bfloat16, float16)")
    if n == 0:
        return [], []
    index = _device([*rms, *ratio, *window], "moments_8bit")
    dev = rms[0].device
    buf, avg, root = bytearray(_MOMENT.size * n), [], []
    with _on(index) as stream:
        for i, (c, r, w) in enumerate(zip(rms, ratio, window)):
            k = c.numel()
            if c.dtype is not torch.uint8 or r.dtype is not torch.int8 or w.dtype is not torch.uint8 or r.numel() != k or w.numel() != (k + WINDOW - 1) // WINDOW:
                raise ValueError(f"moments_8bit: tensor {i}: rms uint8 [n], ratio int8 [n], window uint8 [(n + {WINDOW - 1}) // {WINDOW}] required")
            if not (c.is_contiguous() and r.is_contiguous() and w.is_contiguous()):
                raise ValueError(f"moments_8bit: tensor {i} is not contiguous")
            avg.append(torch.empty(c.shape, dtype=dtype, device=dev))
            root.append(torch.empty(c.shape, dtype=dtype, device=dev))
            _MOMENT.pack_into(buf, _MOMENT.size * i, c.data_ptr(), r.data_ptr(), w.data_ptr(), avg[i].data_ptr(), root[i].data_ptr(), k)
        _lib.check(lib.gsr_adamw_moments(n, _address(buf), betas[0], betas[1], _TYPES[dtype], stream))
    return avg, root


def evict_rows(scores, keep, tensors, recent=0, weights=None, decay=1.0, rms=()):
    """Compacts a map to `keep` of its P rows by accumulated compositing weight.

    scores: float32 [P], accumulated so far; weights: float32 [views, P] or [P], the new views' (compositing_weights), or None:
    score = decay * score + sum of weights.  The last `recent` rows stay whatever their score, and of the others the keep - recent with
    the largest (ties: the lower index; NaN counts as -inf).  tensors: [P, ...] each, of any types; rms: pairs (codes uint8 [P, ...], window)
    of 8-bit moments, re-coded for their new blocks -- exact, but for a root under its new window's sixteen binades, which
    becomes that window's lowest value.  Its ratio (among `tensors`) is copied as it is: the row's next update stays what it was, the exp_avg
    that the bytes stand for grows with the root, and gradients of the row's old size count for little until both have decayed.
    Returns (kept int64 [keep] ascending, scores [keep], [tensor [keep, ...]], [(codes, window)]); the inputs are not written."""
    lib = _lib.load()
    P, keep, recent = scores.numel(), int(keep), int(recent)
    if scores.dim() != 1 or scores.dtype is not torch.float32:
        raise ValueError("evict_rows: scores is float32 [P]")
    if not 0 <= recent <= keep <= P:
        raise ValueError(f"evict_rows: 0 <= recent <= keep <= P required, got recent {recent}, keep {keep}, P {P}")
    if P > 0x7FFFFFFF:
        raise ValueError("evict_rows: at most 2^31 - 1 rows")
    if weights is not None:
        weights = _dense(weights if weights.dim() == 2 else weights.unsqueeze(0))
        if weights.dtype is not torch.float32 or weights.dim() != 2 or weights.shape[1] != P:
            raise ValueError("evict_rows: weights is float32 [views, P] or [P]")
    scores = _dense(scores)
    index = _device([scores, *(() if weights is None else (weights,)), *tensors, *[x for pair in rms for x in pair]], "evict_rows")
    n, size = len(tensors) + len(rms), _ROW.size
    buf, rows, pairs, held = bytearray(size * n), [], [], []
    with _on(index) as stream:
        out = scores.new_empty(keep)
        kept = torch.empty(keep, dtype=torch.int64, device=scores.device)
        at, pack, one = 0, _ROW.pack_into, P == 1
        for t in tensors:
            shape = t.shape
            if not shape or shape[0] != P:
                raise ValueError(f"evict_rows: tensor {len(rows)} has shape {tuple(shape)}, {P} rows wanted")
            if t.is_conj() or one or not t.is_contiguous():
                t = _dense(t)
                held.append(t)
            y = t.new_empty((keep, *shape[1:]))
            rows.append(y)
            pack(buf, at, t.data_ptr(), y.data_ptr(), 0, 0, t.nbytes // P if P else 0)
            at += size
        for c, w in rms:
            k = c.numel()
            if c.dim() < 1 or c.shape[0] != P or c.dtype is not torch.uint8 or w.dtype is not torch.uint8 or w.numel() != (k + WINDOW - 1) // WINDOW:
                raise ValueError(f"evict_rows: rms {len(pairs)}: codes uint8 [P, ...] and their window uint8 required")
            c, w = c.contiguous(), w.contiguous()
            held += (c, w)
            row = k // P if P else 0
            pairs.append((c.new_empty((keep, *c.shape[1:])), w.new_empty((keep * row + WINDOW - 1) // WINDOW)))
            pack(buf, at, c.data_ptr(), pairs[-1][0].data_ptr(), w.data_ptr(), pairs[-1][1].data_ptr(), row)
            at += size
        ws_t, ws = _workspace(lib.gsr_evict_bytes(P), index)
        args = _lib.EvictArgs(P, 0 if weights is None else weights.shape[0], keep, recent, scores.data_ptr(),
                              None if weights is None else weights.data_ptr(), decay, kept.data_ptr(), out.data_ptr(), n, _address(buf),
                              _lib.fixed_buffer_fn(), C.addressof(ws), stream)
        _lib.check(lib.gsr_evict_rows(C.byref(args)))
    return kept, out, rows, pairs


def compositing_weights(raster_settings, means3D, opacities, scales=None, rotations=None, cov3D_precomp=None):
    """float32 [P]: how much each splat contributes to the view that raster_settings (diff_gaussian_rasterization's) describes, the sum over
    pixels of alpha_i T_i -- the derivative of a colour channel's sum by the splat's own colour, so one forward and backward of the
    rasterizer.  What evict_rows accumulates over views."""
    from .rasterizer import GaussianRasterizer
    det = lambda t: None if t is None else t.detach()                                             # noqa: E731
    with torch.enable_grad():
        colors = torch.zeros(means3D.shape[0], 3, dtype=torch.float32, device=means3D.device, requires_grad=True)
        image = GaussianRasterizer(raster_settings)(means3D=det(means3D), means2D=torch.zeros_like(det(means3D)), opacities=det(opacities),
                                                    colors_precomp=colors, scales=det(scales), rotations=det(rotations),
                                                    cov3D_precomp=det(cov3D_precomp))[0]
        ones = torch.zeros_like(image)
        ones[0] = 1.0
        return torch.autograd.grad(image, colors, ones)[0][:, 0].contiguous()


class AdamW(torch.optim.Optimizer):
    """torch.optim.Adam / AdamW for the tensors of a map: `AdamW(groups, lr=0.0, eps=1e-15)` where train.py's
    training_setup (gaussian_splatting/scene/gaussian_model.py:149-167) has `torch.optim.Adam(groups, lr=0.0, eps=1e-15)`.

    weight_decay is decoupled (0, Adam, by default).  state_bits=8 (per group) keeps the moments in two bytes per element; seed is
    that of their stochastic rounding (with the step and a parameter's place among all of the optimiser's).  max_norm clips every step by the
    norm over all groups' gradients, last_norm is then that step's (norm, coefficient) on the device.  With 32 bits the state holds
    "exp_avg" and "exp_avg_sq", shaped like the parameter, so code that indexes, concatenates or replaces them goes on working; with 8 bits
    "rms" and "ratio" are shaped like the parameter and "window" is one byte per 256 elements -- use evict() and append_rows(), which know
    all of them.  "step" is new_clock().

    A group's betas may change between steps, as schedulers do (OneCycleLR): the bias corrections are then torch's, 1 - beta ** t of the current betas, and
    8-bit ratios are read with the betas that they were stored with.  Those are the group's "state_betas", or the state's own "betas" where it has been
    stepped with others.  With 8 bits the first step after such a change cannot be captured, and a captured step is not to be replayed after
    eager ones with other betas."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, state_bits=32, max_norm=None, seed=0):
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError(f"max_norm >= 0 required, got {max_norm}")
        self.max_norm, self.seed, self.last_norm = max_norm, int(seed), None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def __getstate__(self):          # (copies and pickles)
        return dict(super().__getstate__(), max_norm=self.max_norm, seed=self.seed, last_norm=None)

    def add_param_group(self, group):
        super().add_param_group(group)
        g = self.param_groups[-1]
        b1, b2 = g["betas"]
        try:
            if not (torch.is_tensor(g["lr"]) or g["lr"] >= 0.0):
                raise ValueError(f"lr >= 0 required, got {g['lr']}")
            if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
                raise ValueError(f"0 <= beta < 1 required, got {g['betas']}")
            if not g["eps"] >= 0.0 or not g["weight_decay"] >= 0.0:
                raise ValueError(f"eps >= 0 and weight_decay >= 0 required, got {g['eps']}, {g['weight_decay']}")
            if g["state_bits"] not in (32, 8):
                raise ValueError(f"state_bits is 32 or 8, got {g['state_bits']}")
            if g["state_bits"] == 8 and not b1 * b1 < b2:
                raise ValueError(f"8-bit moments need beta1^2 < beta2 (otherwise exp_avg / sqrt(exp_avg_sq) has no bound), got {g['betas']}")
        except ValueError:
            self.param_groups.pop()
            raise
        g.setdefault("state_betas", tuple(g["betas"]))

    def _init_state(self, p, bits):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a parameter's first step cannot be captured (its state would start anew at every replay): step once before")
        st = self.state[p]
        like = lambda dt: torch.zeros(p.shape, dtype=dt, device=p.device)                          # noqa: E731
        if bits == 32:
            st["exp_avg"], st["exp_avg_sq"] = like(torch.float32), like(torch.float32)
        else:
            st["rms"], st["ratio"] = like(torch.uint8), like(torch.int8)
            st["window"] = torch.zeros((p.numel() + WINDOW - 1) // WINDOW, dtype=torch.uint8, device=p.device)
        st["step"] = new_clock(p.device)
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls, grads, moved, place = {}, [], [], -1
        for group in self.param_groups:
            betas, bits, lr, decay = tuple(group["betas"]), group["state_bits"], group["lr"], group["weight_decay"]
            home = group.setdefault("state_betas", betas)
            call = calls.setdefault((bits, betas, group["eps"]), [])
            for p in group["params"]:
                place += 1          # (of a parameter, whichever others are stepped and in how many calls: its random bits are its own)
                g = p.grad
                if g is None:
                    continue
                if g.layout is not torch.strided:
                    raise RuntimeError("AdamW does not support sparse gradients")
                st = self.state[p] if p in self.state else None
                if not st:
                    _device((p,), "AdamW")
                    st = self._init_state(p, bits)
                    if betas != home:
                        st["betas"] = betas
                was = st.get("betas", home)
                if was != betas:
                    if bits == 8 and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: the first 8-bit step with other betas cannot be captured (every replay would read the ratios with the old ones): step once before")
                    moved.append((st, betas, home))
                call.append((p, g, st["exp_avg"], st["exp_avg_sq"], st["step"], lr, decay) if bits == 32 else
                            (p, g, st["rms"], st["ratio"], st["step"], lr, decay, st["window"], (was, place)))
                grads.append(g)
        if not grads:
            return loss
        clip = None if self.max_norm is None else grad_norm(grads, self.max_norm)
        # (made whole or not at all: everything is checked before anything is launched)
        packed = []
        for (bits, betas, eps), call in calls.items():
            if not call:
                continue
            p, g, a, b, clock, lr, decay, *coded = zip(*call)
            window, origin = coded or (None, None)
            if coded and not moved and origin[-1][1] == len(p) - 1:
                origin = None          # (this step's betas, places in the list)
            packed.append(_pack(bits, "AdamW", p, g, a, b, window, clock, lr, betas, eps, decay, clip, self.seed, origin))
        if len(packed) > 1 or moved:
            for args, origins, *_ in packed:
                _lib.check(_lib.load().gsr_adamw_check(C.byref(args), _address(origins)))
        for st, betas, home in moved:
            # torch's corrections: 1 - beta ** t, of this step's betas
            for k in (0, 1):
                torch.pow(betas[k], st["step"][2], out=st["step"][k])
        for call in packed:
            _launch(call)
        for st, betas, home in moved:
            st["betas"] = betas
            if betas == home:
                del st["betas"]
        if clip is not None:
            self.last_norm = clip
        return loss

    def load_state_dict(self, state_dict):
        """Takes its own state_dict() and torch.optim.Adam's / AdamW's (32-bit groups): states keep their types whatever the parameter's.
        weight_decay is decoupled here: a group of torch's that has one must say that its is ("decoupled_weight_decay"; torch's AdamW does)."""
        own, given = self.param_groups, state_dict["param_groups"]
        bits = [g.get("state_bits", own[k]["state_bits"]) if k < len(own) else 32 for k, g in enumerate(given)]
        for b, g in zip(bits, given):
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("load_state_dict: amsgrad and maximize are not supported")
            if g.get("weight_decay") and not g.get("decoupled_weight_decay", "state_bits" in g):
                raise ValueError("load_state_dict: a group's weight_decay is not decoupled, or its state_dict does not say (if it is, set the group's decoupled_weight_decay to True)")
            wanted = {"exp_avg", "exp_avg_sq", "step"} if b == 32 else {"rms", "ratio", "window", "step"}
            for i in g["params"]:
                if i in state_dict["state"] and not wanted <= set(state_dict["state"][i]):
                    raise ValueError(f"load_state_dict: a group with {b}-bit moments got the state {sorted(state_dict['state'][i])}")
        super().load_state_dict(state_dict)
        for b, g, old in zip(bits, self.param_groups, given):
            for k in ("amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay"):
                g.pop(k, None)          # (torch.optim.Adam's own options)
            g["state_bits"] = b
            g["betas"] = tuple(g["betas"])
            g["state_betas"] = tuple(g.get("state_betas", g["betas"]))
            for i, p in zip(old["params"], g["params"]):
                if i not in state_dict["state"]:
                    continue
                # (the base class casts every state to the parameter's type)
                st = {k: v.detach().to(device=p.device, copy=True) if torch.is_tensor(v) else v for k, v in state_dict["state"][i].items()}
                if not torch.is_tensor(st["step"]) or st["step"].numel() == 1:
                    t = float(st["step"])
                    st["step"] = torch.tensor([g["betas"][0] ** t, g["betas"][1] ** t, t, 0.0], dtype=torch.float64, device=p.device)
                st["step"] = st["step"].double()
                if b == 32:
                    st["exp_avg"], st["exp_avg_sq"] = st["exp_avg"].float(), st["exp_avg_sq"].float()
                self.state[p] = st

    def _replace(self, old, data, states):
        new = torch.nn.Parameter(data, requires_grad=old.requires_grad)
        st = self.state.pop(old, None)
        if st:
            self.state[new] = dict(st, **states)
        for g in self.param_groups:
            g["params"] = [new if p is old else p for p in g["params"]]

    @torch.no_grad()
    def evict(self, scores, keep, recent=0, weights=None, decay=1.0, extra=()):
        """evict_rows over every parameter, its state and `extra` (other [P, ...] tensors, e.g. max_radii2D): the groups hold new
        Parameters afterwards, without gradients.  Returns (kept, scores, [extra])."""
        params = [p for g in self.param_groups for p in g["params"]]
        names = [[k for k in ("exp_avg", "exp_avg_sq", "ratio") if k in self.state.get(p, {})] for p in params]
        coded = [p for p in params if "rms" in self.state.get(p, {})]
        rows = [p.detach() for p in params] + [self.state[p][k] for p, ks in zip(params, names) for k in ks] + list(extra)
        kept, out, rows, pairs = evict_rows(scores, keep, rows, recent, weights, decay, [(self.state[p]["rms"], self.state[p]["window"]) for p in coded])
        rest, pairs = iter(rows[len(params):]), dict(zip(map(id, coded), pairs))
        for p, data, ks in zip(params, rows, names):
            states = {k: next(rest) for k in ks}
            if id(p) in pairs:
                states["rms"], states["window"] = pairs[id(p)]
            self._replace(p, data, states)
        return kept, out, list(rest)

    @torch.no_grad()
    def append_rows(self, new):
        """Adds rows to every parameter (cat_tensors_to_optimizer, gaussian_model.py:307-328): `new` is one tensor per parameter, in the groups'
        order; the newcomers' moments are zero, the step counts go on.  The groups hold new Parameters afterwards, without gradients."""
        params = [p for g in self.param_groups for p in g["params"]]
        if len(new) != len(params):
            raise ValueError(f"append_rows: {len(new)} tensors for {len(params)} parameters")
        for p, x in zip(params, new):
            if x.shape[1:] != p.shape[1:] or x.dim() != p.dim():
                raise ValueError(f"append_rows: rows of shape {tuple(x.shape)} for a parameter of shape {tuple(p.shape)}")
        for p, x in zip(params, new):
            data = torch.cat((p.detach(), x.detach().to(device=p.device, dtype=p.dtype)))
            states = {}
            for k, v in self.state.get(p, {}).items():
                if k in ("exp_avg", "exp_avg_sq", "rms", "ratio"):
                    states[k] = torch.cat((v, v.new_zeros(x.shape)))
                elif k == "window":
                    states[k] = torch.cat((v, v.new_zeros((data.numel() + WINDOW - 1) // WINDOW - v.numel())))
            self._replace(p, data, states)
