"""AdamW over all parameters of a group in one launch, with 32-bit or 8-bit states."""

import torch

from .. import _native as nat

_CODE = torch.float8_e4m3fn
_BLOCK = 256  # values that share a scale; every tensor's states start on such a boundary


class _Bucket:
    """The parameters of one group with one type on one device, and their flat states."""

    def __init__(self, params, bits):
        self.params = params
        self.device, self.dtype = params[0].device, params[0].dtype
        nat.require_cuda(params[0])
        if self.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError("parameters must be float32, bfloat16 or float16, got {}".format(
                self.dtype))
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("take one step before a step is captured: a replay would zero the "
                               "states that the captured one makes")
        self.sizes = [p.numel() for p in params]
        at = sum(-(-n // _BLOCK) * _BLOCK for n in self.sizes)
        dev = self.device
        f32 = dict(dtype=torch.float32, device=dev)
        self.step = torch.zeros(2, dtype=torch.int32, device=dev)
        if bits == 32:
            self.state = {"exp_avg": torch.zeros(at, **f32), "exp_avg_sq": torch.zeros(at, **f32)}
        else:
            code = dict(dtype=_CODE, device=dev)
            self.state = {"exp_avg": torch.zeros(at, **code),
                          "exp_avg_scale": torch.zeros(at // _BLOCK, **f32),
                          "exp_avg_sqrt": torch.zeros(at, **code),
                          "exp_avg_sqrt_scale": torch.zeros(at // _BLOCK, **f32)}
        self.bits = bits

    # pickle takes no float8 tensors: codes travel as bytes
    def __getstate__(self):
        return {**self.__dict__, "state": {k: v.view(torch.uint8) if v.dtype == _CODE else v
                                           for k, v in self.state.items()}}

    def __setstate__(self, saved):
        self.__dict__.update(saved)
        self.state = {k: v.view(_CODE) if v.dtype == torch.uint8 else v
                      for k, v in self.state.items()}

    def buffers(self):
        """First moments and their scales, second moments and theirs."""
        s = self.state
        if self.bits == 32:
            return s["exp_avg"], None, s["exp_avg_sq"], None
        return tuple(s[k] for k in ("exp_avg", "exp_avg_scale", "exp_avg_sqrt",
                                    "exp_avg_sqrt_scale"))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) in one kernel launch per group and type.

    Args:
        params: Parameters or groups of them: float32, bfloat16 or float16 CUDA tensors.
        lr: Learning rate, a number or a one-element float32 CUDA tensor.  A step captured in a
            CUDA graph (after one that was not) reads the tensor at each replay; a number is
            captured as it is.
        betas, eps, weight_decay: As in ``torch.optim.AdamW``.
        state_bits: 32, or 8: the first moment and the root of the second as e4m3 codes with a
            float32 scale per 256 values, rounded stochastically.
        seed: Of that rounding; one seed gives one result.

    The states of a group's parameters lie in flat buffers (``flat_state``), made at the first step:
    from then on the group keeps its parameters, and they their sizes.  The step count is the
    group's (of the parameters of one type in it) and lives on the device; a parameter without a
    gradient is left out of a step, and a step in which none has one is not counted.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits=32, seed=0):
        if not isinstance(lr, torch.Tensor) and not lr >= 0:
            raise ValueError("lr must be >= 0")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("betas must be in [0, 1)")
        if not eps >= 0:
            raise ValueError("eps must be >= 0")
        if not weight_decay >= 0:
            raise ValueError("weight_decay must be >= 0")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self._bits, self._seed, self._buckets = state_bits, int(seed), {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        """Copies and pickles keep the states and whose they are, not only the groups."""
        return {**super().__getstate__(), "_bits": self._bits, "_seed": self._seed,
                "_buckets": self._buckets}

    def _group_buckets(self, index):
        """Made at the first step, when the parameters are where they will stay."""
        group = self.param_groups[index]["params"]
        if index not in self._buckets:
            kinds = {}
            for p in group:
                kinds.setdefault((p.device, p.dtype), []).append(p)
            self._buckets[index] = tuple(group), [_Bucket(ps, self._bits) for ps in kinds.values()]
        members, have = self._buckets[index]
        if not nat.host().same_objects(members, group):
            raise ValueError("the parameters of group {} are not those that its states were made "
                             "for; new ones come with add_param_group".format(index))
        return have

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        launches = []
        for index, group in enumerate(self.param_groups):
            lr = group["lr"]
            on_device = isinstance(lr, torch.Tensor)
            for b in self._group_buckets(index):
                m, ms, v, vs = b.buffers()
                launches.append((b.params, b.sizes, self._bits, m, ms, v, vs, b.step,
                                 0.0 if on_device else lr, lr if on_device else None,
                                 *group["betas"], group["eps"], group["weight_decay"],
                                 self._seed & 0xFFFFFFFF))
        host = nat.host()
        if len(launches) > 1:  # a refused step changes nothing
            for args in launches:
                host.adamw_check(*args)
        for args in launches:
            host.adamw_step(*args)
        return loss

    def flat_state(self, index=0):
        """The flat state buffers of bucket ``index`` (groups in order, a bucket for each type in
        them): ``exp_avg`` and ``exp_avg_sq``, or in 8 bits ``exp_avg`` and ``exp_avg_sqrt`` with
        their ``*_scale``.  Each tensor's states start on a multiple of 256 values, in the order
        of the parameters."""
        buckets = [b for i in range(len(self.param_groups)) for b in self._group_buckets(i)]
        return dict(buckets[index].state)

    def state_dict(self):
        """Hyperparameters by group, and the flat states of every bucket: the live tensors, their
        step count among them, as ``torch.optim`` gives them."""
        out = super().state_dict()
        out["state_bits"] = self._bits
        out["seed"] = self._seed
        out["buckets"] = [{"step": b.step[:1], **b.state}
                          for i in range(len(self.param_groups)) for b in self._group_buckets(i)]
        return out

    def load_state_dict(self, state_dict):
        if state_dict.get("state_bits") != self._bits:
            raise ValueError("the saved states have {} bits, this optimizer's {}".format(
                state_dict.get("state_bits"), self._bits))
        # all is checked before anything changes (the groups by the base class, first thing)
        mine = [b for i in range(len(self.param_groups)) for b in self._group_buckets(i)]
        saved = state_dict["buckets"]
        if len(mine) != len(saved) or any(k not in s or v.shape != s[k].shape
                                          for b, s in zip(mine, saved)
                                          for k, v in {**b.state, "step": b.step[:1]}.items()):
            raise ValueError("the saved states belong to other parameters")
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        self._seed = int(state_dict["seed"])
        for b, s in zip(mine, saved):
            b.step[:1].copy_(s["step"])
            for k, v in b.state.items():
                v.copy_(s[k])
