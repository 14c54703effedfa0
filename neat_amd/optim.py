"""AdamW over the adapted LayerNorm parameters as ONE kernel launch.

Same update rule and defaults as ``torch.optim.AdamW`` (reference main_TTA.py:271: lr = tta_init_lr,
weight_decay = tta_wd, betas (0.9, 0.999), eps 1e-8; state persists across batches).  The 48 (ViT-B-32)
parameter tensors are re-pointed at construction to views of one flat fp32 buffer, their ``.grad`` to
views of a flat gradient buffer, so ``step()`` is a single ``neat_adamw_flat`` launch instead of 48
small ones and a data-parallel gradient all-reduce is one collective over ``flat_grad``.

``MultiTensorAdamW`` applies the same rule to any number of tensors that stay where they are -- float32 or bfloat16, several
parameter groups, gradients that come and go -- with moments in 32 or in 8 bits (``neat_adamw_multi``).
"""
from __future__ import annotations

import array
import itertools
import operator

import torch

from . import lib, ops


class AdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        params = list(params)
        if not params:
            raise ValueError("AdamW: empty parameter list")
        if any(isinstance(p, dict) for p in params):
            raise ValueError("neat_amd.optim.AdamW supports a single parameter group")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        dev = params[0].device
        if dev.type != "cuda":
            raise RuntimeError("neat_amd.optim.AdamW: parameters must be on the GPU")
        n = sum(p.numel() for p in params)
        self.flat_param = torch.empty(n, dtype=torch.float32, device=dev)
        # two spare floats behind the gradients: the data-parallel step sends its two row-summed loss terms with the
        # gradient in ONE all-reduce over grad_buf
        self.grad_buf = torch.zeros(n + 2, dtype=torch.float32, device=dev)
        self.flat_grad = self.grad_buf[:n]
        self.exp_avg = torch.zeros(n, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(n, dtype=torch.float32, device=dev)
        self.step_count = 0
        off = 0
        for p in params:
            k = p.numel()
            self.flat_param[off:off + k].copy_(p.detach().reshape(-1))
            p.data = self.flat_param[off:off + k].view_as(p)
            p.grad = self.flat_grad[off:off + k].view_as(p)
            off += k

    @torch.no_grad()
    def step(self, closure=None):
        g = self.param_groups[0]
        # the parameters and their gradients must still be the views made in __init__: a later model.to()/.float()/
        # .cuda() re-creates p.data, and p.grad = None drops the gradient view -- the step would then update buffers
        # nobody reads.  Two pointer comparisons per step (first and last parameter).
        off_last = self.flat_param.numel() - g["params"][-1].numel()
        for p, off in ((g["params"][0], 0), (g["params"][-1], off_last)):
            if (p.data_ptr() != self.flat_param[off:].data_ptr() or p.grad is None
                    or p.grad.data_ptr() != self.flat_grad[off:].data_ptr()):
                raise RuntimeError("neat_amd.optim.AdamW: a parameter (or its .grad) no longer aliases the optimizer's flat "
                                   "buffers -- build the optimizer AFTER moving/casting the model, and clear gradients "
                                   "with optimizer.zero_grad() rather than p.grad = None")
        self.step_count += 1
        ops.adamw_flat(self.flat_param, self.flat_grad, self.exp_avg, self.exp_avg_sq, self.step_count, g["lr"],
                       g["betas"][0], g["betas"][1], g["eps"], g["weight_decay"])

    def zero_grad(self, set_to_none: bool = False):
        # gradients are views of flat_grad and must stay attached; the backward overwrites them
        self.flat_grad.zero_()


_grad_of = operator.attrgetter("grad")


def _at(a):
    return a.buffer_info()[0]


class MultiTensorAdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` over float32 / bfloat16 parameters of any sizes, one launch per 96 tensors.

    ``state_bits=32``: the moments are ``exp_avg`` and ``exp_avg_sq``, float32 [blocks, 256]; every parameter owns
    ceil(numel / 256) blocks, in parameter order.  ``state_bits=8``: ``exp_avg`` and ``exp_avg_root`` (the SQUARE ROOT of
    the second moment) are e4m3 numbers [blocks, 256], each block times its power of two ``exp_avg_scale`` /
    ``exp_avg_root_scale`` [blocks]: 2 bytes an element instead of 8.  ``moments(p)`` gives one parameter's as it would be
    in 32 bits.  A parameter whose ``.grad`` is None is left alone and its step count stays (as in torch).

    The host looks at every tensor on every step (0.03 us each; 0.5 us in a step where a gradient is missing or not contiguous)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        if state_bits not in (32, 8):
            raise ValueError(f"MultiTensorAdamW: state_bits must be 32 or 8, got {state_bits}")
        self._ready = False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        for g in self.param_groups:
            self._check_group(g)
        ps = [p for g in self.param_groups for p in g["params"]]
        if not ps:
            raise ValueError("MultiTensorAdamW: empty parameter list")
        if len(set(map(id, ps))) != len(ps):
            raise ValueError("MultiTensorAdamW: a parameter is listed twice")
        if ps[0].device.type != "cuda" or len(set(map(torch.Tensor.get_device, ps))) != 1:
            raise RuntimeError("MultiTensorAdamW: parameters must be on one GPU")
        dtypes = [p.dtype for p in ps]
        if not set(dtypes) <= {torch.float32, torch.bfloat16}:
            raise RuntimeError(f"MultiTensorAdamW: parameters must be float32 or bfloat16, got {set(dtypes)}")
        if not all(map(torch.Tensor.is_contiguous, ps)):
            raise RuntimeError("MultiTensorAdamW: parameters must be contiguous")
        at = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in ps if p.numel())
        if any(b[0] < a[1] for a, b in zip(at, at[1:])):
            raise ValueError("MultiTensorAdamW: two parameters share memory (they would be updated at once)")
        lib.step_list()                              # a missing helper is an error here, not in the first step
        self._lay_out(ps, state_bits)
        self._ready = True

    def _lay_out(self, ps, state_bits, buffers=None):
        """The moments of ``ps`` (new ones, or ``buffers``), and what a step needs to know of them."""
        self.state_bits, self.device = state_bits, ps[0].device
        # by position in the list of all parameters: sizes, first blocks of the moments
        self._params, self._numel = ps, list(map(torch.Tensor.numel, ps))
        ends = list(itertools.accumulate([-(-n // ops.ADAMW_BLOCK) for n in self._numel]))
        self._first, blocks = [0] + ends[:-1], ends[-1]
        # per group and type, what one call of the library updates: [group, type, positions, parameters, layout, step counts]
        self._lists, at = [], 0
        for i, g in enumerate(self.param_groups):
            here = range(at, at + len(g["params"]))
            at = here.stop
            for dt in (torch.float32, torch.bfloat16):
                pos = [k for k in here if ps[k].dtype == dt]
                if pos:
                    self._lists.append([i, dt, pos, [ps[k] for k in pos], self._layout(pos), array.array("i", [0] * len(pos))])
        if buffers is None:
            dt = torch.uint8 if state_bits == 8 else torch.float32
            buffers = [torch.zeros(blocks, ops.ADAMW_BLOCK, dtype=dt, device=self.device) for _ in range(2)]
            buffers += [torch.ones(blocks, device=self.device) for _ in range(2)] if state_bits == 8 else []
        self._m, self._v, self._ms, self._vs = [*buffers, None, None][:4]
        # e4m3 views of the codes (the same memory)
        self.exp_avg = self._m.view(torch.float8_e4m3fn) if state_bits == 8 else self._m
        if state_bits == 8:
            self.exp_avg_root, self.exp_avg_scale, self.exp_avg_root_scale = self._v.view(torch.float8_e4m3fn), self._ms, self._vs
        else:
            self.exp_avg_sq = self._v

    def __getstate__(self):
        return dict(super().__getstate__(), _held=(self.state_bits, self._buffers(), self._step_counts()))

    def __setstate__(self, state):
        """For copies and pickles; torch calls it from load_state_dict too, without the moments."""
        held = state.get("_held")
        super().__setstate__({k: v for k, v in state.items() if k != "_held"})
        if held is not None:
            bits, buffers, steps = held
            self._lay_out([p for g in self.param_groups for p in g["params"]], bits, buffers)
            self._set_step_counts(steps)
            self._ready = True

    def _layout(self, pos):
        """(sizes, the same as a C array, first blocks of the moments as a C array)."""
        sizes = [self._numel[k] for k in pos]
        return sizes, array.array("q", sizes), array.array("q", [self._first[k] for k in pos])

    @staticmethod
    def _check_group(g):
        b1, b2 = g["betas"]
        if not 0.0 <= b1 < 1.0 or not 0.0 <= b2 < 1.0:
            raise ValueError(f"MultiTensorAdamW: betas must lie in [0, 1), got {g['betas']}")
        if g["lr"] < 0.0 or g["eps"] < 0.0 or g["weight_decay"] < 0.0:
            raise ValueError("MultiTensorAdamW: lr, eps and weight_decay must not be negative")

    def add_param_group(self, group):
        if getattr(self, "_ready", False):
            raise RuntimeError("MultiTensorAdamW: the moments are laid out when it is built; pass all groups then")
        super().add_param_group(group)

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # every list is looked at before the first one is launched: a step that is refused has changed nothing
        calls = []
        for i, dt, pos, ps, layout, steps in self._lists:
            group = self.param_groups[i]
            b1, b2 = group["betas"]
            rates = float(group["lr"]), float(b1), float(b2), float(group["eps"]), float(group["weight_decay"])
            n, (_, sizes_c, blocks_c) = len(ps), layout
            p_c, g_c, now = array.array("Q", bytes(8 * n)), array.array("Q", bytes(8 * n)), array.array("i", bytes(4 * n))
            # the common step: every parameter has a gradient, and all are as they were laid out
            if lib.step_list()(ps, n, _at(sizes_c), dt == torch.bfloat16, self.device.index, _at(steps), _at(p_c), _at(g_c), _at(now)):
                calls.append((n, p_c, g_c, sizes_c, blocks_c, now, dt, rates, steps, None, ps, None))
                continue
            grads = list(map(_grad_of, ps))
            at = [k for k, g in enumerate(grads) if g is not None]
            if at:
                sizes, sizes_c, blocks_c = self._layout([pos[k] for k in at])
                some = [ps[k] for k in at]
                if some[0].device != self.device:
                    raise RuntimeError(f"MultiTensorAdamW: parameters must stay on {self.device}, where the moments are")
                p_c, g_c, held = ops._adamw_addresses(some, [grads[k] for k in at], sizes)
                now = array.array("i", [steps[k] + 1 for k in at])
                calls.append((len(at), p_c, g_c, sizes_c, blocks_c, now, some[0].dtype, rates, steps, at, some, held))
        for n, p_c, g_c, sizes_c, blocks_c, now, dt, rates, steps, at, ps, _ in calls:
            ops._adamw_launch(self.device, n, p_c, g_c, sizes_c, blocks_c, now, dt, self._m, self._v, self._ms, self._vs, *rates)
            lib.written()(ps)                        # a backward pass that saved them is to raise an error, as with torch's AdamW
            if at is None:
                steps[:] = now
            else:
                for k, c in zip(at, now):
                    steps[k] = c
        return loss

    def _step_counts(self):
        """Step counts by position."""
        counts = [0] * len(self._params)
        for _, _, pos, _, _, steps in self._lists:
            for k, n in zip(pos, steps):
                counts[k] = n
        return counts

    def moments(self, p):
        """(exp_avg, exp_avg_sq) of one parameter in float32, in its shape, and its step count."""
        k = next((k for k, q in enumerate(self._params) if q is p), None)
        if k is None:
            raise ValueError("MultiTensorAdamW: not one of this optimizer's parameters")
        n, lo = self._numel[k], self._first[k]
        rows = slice(lo, lo - (-n // ops.ADAMW_BLOCK))
        m, v = self.exp_avg[rows].float(), (self.exp_avg_root if self.state_bits == 8 else self._v)[rows].float()
        if self.state_bits == 8:
            m, v = m * self._ms[rows, None], (v * self._vs[rows, None]) ** 2
        return m.reshape(-1)[:n].view(p.shape), v.reshape(-1)[:n].view(p.shape), self._step_counts()[k]

    def _buffers(self):
        return [t for t in (self._m, self._v, self._ms, self._vs) if t is not None]

    def state_dict(self):
        d = super().state_dict()
        d["state"] = {"state_bits": self.state_bits, "numels": list(self._numel), "steps": self._step_counts(),
                      "buffers": self._buffers()}
        return d

    def _set_step_counts(self, steps):
        for _, _, pos, _, _, held in self._lists:
            held[:] = array.array("i", [int(steps[k]) for k in pos])

    def load_state_dict(self, state_dict):
        st = state_dict["state"]
        if st.get("state_bits") != self.state_bits or st["numels"] != self._numel:
            raise ValueError("MultiTensorAdamW: the state belongs to other parameters or another state_bits")
        mine, given = self._buffers(), list(st["buffers"])
        if len(st["steps"]) != len(self._numel) or [(t.shape, t.dtype) for t in given] != [(t.shape, t.dtype) for t in mine]:
            raise ValueError("MultiTensorAdamW: the state's moments are not laid out as this optimizer's")
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        for dst, src in zip(mine, given):
            dst.copy_(src)
        self._set_step_counts(st["steps"])
