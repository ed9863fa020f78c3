"""Training-step plumbing for the hot path: flat parameter/gradient bucket, fused clip + Adam (HIP),
one RCCL all-reduce per step.

Replaces, for the data-parallel path, nn.DataParallel's per-step broadcast/scatter/gather/reduce
(src/hl_modules/distance_based_hl_module.py:34-35) and PLModule.reset_grad/backprop (:430-441):
one process per GPU, identical replicas, ONE all-reduce over a single flat fp32 gradient buffer
(2.0 MB big / 0.9 MB small), then clip_grad_norm_ semantics and Adam on every rank.
"""
import torch

from . import ops
from .forms import bump_weight_epoch


class FlatBucket:
    """All parameters of `module` re-pointed into one contiguous fp32 buffer; grads likewise."""

    def __init__(self, module):
        self.params = [p for p in module.parameters() if p.requires_grad]
        dev = self.params[0].device
        n = sum(p.numel() for p in self.params)
        # 16-byte align every parameter so the HIP kernels can use 128-bit loads on weight rows
        offs, off = [], 0
        for p in self.params:
            offs.append(off)
            off += (p.numel() + 3) // 4 * 4
        self.numel = off
        self.flat = torch.zeros(off, device=dev, dtype=torch.float32)
        self.grad = torch.zeros(off, device=dev, dtype=torch.float32)
        for p, o in zip(self.params, offs):
            self.flat[o:o + p.numel()].copy_(p.data.reshape(-1))
            p.data = self.flat[o:o + p.numel()].view(p.shape)
            p.grad = self.grad[o:o + p.numel()].view(p.shape)
            p._sb_flat_grad = True          # functional._GradTargets: the HIP reductions may accumulate into .grad directly
        self.offsets = offs
        self.n_params = n

    def zero_grad(self):
        self.grad.zero_()


class FusedAdam:
    """torch.optim.Adam(lr, betas, eps) semantics (no weight decay / amsgrad) over a FlatBucket, with
    clip_grad_norm_(max_norm=grad_clip) folded in.  `lr` may be changed between steps (schedulers)."""

    def __init__(self, bucket, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, amsgrad=False):
        if weight_decay or amsgrad:
            raise NotImplementedError("weight_decay / amsgrad are not used by any shipped config")
        self.bucket, self.lr, self.betas, self.eps = bucket, lr, betas, eps
        self.m = torch.zeros_like(bucket.flat)
        self.v = torch.zeros_like(bucket.flat)
        self.step_count = 0
        self.sumsq = torch.zeros(1, device=bucket.flat.device, dtype=torch.float32)
        # optimiser steps the kernel turned into no-ops because the watchdog word of the guarded schedules was set (a bounded
        # wait of that step's launches gave up: garbage gradients).  Read with the word itself (ops.check_sched_status*).
        self.skipped = torch.zeros(1, device=bucket.flat.device, dtype=torch.int32)
        self.param_groups = [{"lr": lr}]        # scheduler-facing view (get_current_lr, hl_module:158-160)

    def step(self, grad_clip=None, world_size=1):
        """grads already SUMMED over ranks; they are scaled by 1/world_size here."""
        b = self.bucket
        self.step_count += 1
        lr = self.param_groups[0]["lr"]
        clip = float(grad_clip) if grad_clip else 0.0
        if clip > 0:
            ops.sumsq(b.grad, self.sumsq, accumulate=False)
        ops.adam_step(b.flat, b.grad, self.m, self.v, lr, self.betas[0], self.betas[1], self.eps, self.step_count,
                      gscale=1.0 / world_size, clip=clip, sumsq_buf=self.sumsq, skipped=self.skipped)
        bump_weight_epoch()       # the kernel wrote the parameters behind torch's version counters: weight forms are stale

    def state_tensors(self):
        """what makes two replicas' optimisers the same, beside step_count and lr (broadcast_replica)"""
        return [self.m, self.v]

    def state_dict(self):
        """torch.optim.Adam.state_dict() layout (what the reference's dump_state stores under 'optimizer',
        hl_module:141-156): per-parameter {step, exp_avg, exp_avg_sq} indexed in model.parameters() order, sliced out of
        the flat moment buffers, plus one param_group -- so the reference's load_state can resume from our last.pt."""
        b = self.bucket
        state = {}
        if self.step_count > 0:
            for i, (p, o) in enumerate(zip(b.params, b.offsets)):
                n = p.numel()
                state[i] = {"step": torch.tensor(float(self.step_count)),
                            "exp_avg": self.m[o:o + n].view(p.shape).clone(),
                            "exp_avg_sq": self.v[o:o + n].view(p.shape).clone()}
        group = {"lr": self.param_groups[0]["lr"], "betas": tuple(self.betas), "eps": self.eps, "weight_decay": 0,
                 "amsgrad": False, "maximize": False, "foreach": None, "capturable": False, "differentiable": False,
                 "fused": None, "decoupled_weight_decay": False, "params": list(range(len(b.params)))}
        return {"state": state, "param_groups": [group]}

    def load_state_dict(self, sd):
        """Accepts torch.optim.Adam's layout (a reference last.pt / best.pt) and this class's round-1 private layout
        {m, v, step, lr}."""
        b = self.bucket
        if "m" in sd and "param_groups" not in sd:                  # round-1 layout
            self.m.copy_(sd["m"])
            self.v.copy_(sd["v"])
            self.step_count = int(sd["step"])
            self.param_groups[0]["lr"] = sd["lr"]
            return
        groups = sd["param_groups"]
        order = [i for g in groups for i in g["params"]]
        if len(order) != len(b.params):
            raise ValueError(f"optimizer state covers {len(order)} parameters, the model has {len(b.params)}")
        g0 = groups[0]
        if g0.get("weight_decay", 0) or g0.get("amsgrad", False) or g0.get("maximize", False):
            raise NotImplementedError("weight_decay / amsgrad / maximize optimizer states are not supported")
        self.m.zero_()
        self.v.zero_()
        steps = set()
        for slot, (p, o) in zip(order, zip(b.params, b.offsets)):
            st = sd["state"].get(slot)
            if st is None:
                continue
            if tuple(st["exp_avg"].shape) != tuple(p.shape):
                raise ValueError(f"optimizer state {slot}: shape {tuple(st['exp_avg'].shape)} != parameter {tuple(p.shape)}")
            n = p.numel()
            self.m[o:o + n].copy_(st["exp_avg"].reshape(-1))
            self.v[o:o + n].copy_(st["exp_avg_sq"].reshape(-1))
            steps.add(int(float(st["step"])))
        if len(steps) > 1:
            raise ValueError(f"per-parameter Adam step counts differ ({sorted(steps)}): one shared step is supported")
        self.step_count = steps.pop() if steps else 0
        self.param_groups[0]["lr"] = g0["lr"]
        self.betas, self.eps = tuple(g0.get("betas", self.betas)), g0.get("eps", self.eps)


class FusedAdamW:
    """torch.optim.AdamW(lr, betas, eps, weight_decay) semantics (no amsgrad) over a FlatBucket or any list of parameters -- float32,
    or bfloat16 / float16 with an fp32 master copy -- in one launch for 112 tensors (ops.adamw_step), with
    clip_grad_norm_(max_norm=grad_clip) folded in.

    state_bits = 8 keeps exp_avg and exp_avg_sq as 8-bit floats with a power-of-two scale for every 256 elements: 2 bytes a parameter
    instead of 8; `seed` is their rounding's.  A parameter whose .grad is None is left alone in that step; the bias
    corrections count the optimiser's steps, for all parameters alike.
    16-bit parameters that something else has written (a checkpoint, say) are taken over into the master copy by sync_master().
    capturable = True keeps step and lr on the device, so that a captured step counts on at every replay; `lr` is then taken over
    from param_groups by every step outside a capture, or by sync_lr()."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, state_bits=32, seed=0,
                 capturable=False):
        if amsgrad:
            raise NotImplementedError("amsgrad is not used by any shipped config")
        self.params = list(params.params if isinstance(params, FlatBucket) else params)
        if not self.params:
            raise ValueError("FusedAdamW: no parameters")
        self.lr, self.betas, self.eps, self.weight_decay, self.seed = lr, tuple(betas), eps, weight_decay, int(seed)
        self.state = ops.adamw_state(self.params, state_bits)
        self.starts = [b * ops.L.ADAMW_BLOCK for b in ops.adamw_blocks([p.numel() for p in self.params])]
        dev = self.params[0].device
        self.capturable = bool(capturable)
        self._step = torch.zeros(1, dtype=torch.int32, device=dev) if capturable else 0
        self._lr_dev = torch.full((1,), float(lr), dtype=torch.float32, device=dev) if capturable else None
        self.skipped = torch.zeros(1, device=dev, dtype=torch.int32)       # as FusedAdam's
        self.param_groups = [{"lr": lr}]

    @property
    def step_count(self):
        """(synchronises where capturable)"""
        return int(self._step)

    @step_count.setter
    def step_count(self, n):
        if self.capturable:
            self._step.fill_(int(n))
        else:
            self._step = int(n)

    def sync_master(self):
        """the parameters' present values to their fp32 master copies"""
        if "master" in self.state:
            for p, o in zip(self.params, self.starts):
                self.state["master"][o:o + p.numel()].copy_(p.detach().reshape(-1))

    def sync_lr(self):
        """param_groups' lr to the device, for graphs that are replayed"""
        if self.capturable:
            self._lr_dev.fill_(float(self.param_groups[0]["lr"]))

    def step(self, grad_clip=None, world_size=1):
        """grads already SUMMED over ranks; they are scaled by 1/world_size here."""
        if self.capturable:
            if not torch.cuda.is_current_stream_capturing():
                self.sync_lr()
            self._step.add_(1)
            step, lr = self._step, self._lr_dev
        else:
            step, lr = self._step + 1, self.param_groups[0]["lr"]
        try:
            with torch.no_grad():
                ops.adamw_step(self.params, [p.grad for p in self.params], self.state, step, lr=lr, betas=self.betas, eps=self.eps,
                               weight_decay=self.weight_decay, gscale=1.0 / world_size, clip=float(grad_clip) if grad_clip else 0.0,
                               seed=self.seed, skipped=self.skipped)
        except ops.L.SoundBubbleHipError:
            if self.capturable:      # (refused: the step does not count)
                self._step.sub_(1)
            raise
        if not self.capturable:
            self._step = step
        bump_weight_epoch()

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if p.grad is not None:
                if set_to_none and not getattr(p, "_sb_flat_grad", False):
                    p.grad = None
                else:
                    p.grad.zero_()

    def state_tensors(self):
        return [t if t.dtype == torch.float32 else t.view(torch.uint8) for t in self.state.values()]

    def state_dict(self):
        """torch.optim.AdamW.state_dict() layout, as FusedAdam's; 8-bit states as the float32 values they stand for, and
        `master_param` for a 16-bit parameter"""
        state, n = {}, self.step_count
        if n > 0:
            values = ops.adamw_state_values(self.state)
            if "master" in self.state:
                values["master_param"] = self.state["master"]
            for i, (p, o) in enumerate(zip(self.params, self.starts)):
                state[i] = {"step": torch.tensor(float(n)), **{k: v[o:o + p.numel()].view(p.shape).clone() for k, v in values.items()
                                                               if k != "master_param" or p.dtype != torch.float32}}
        group = {"lr": self.param_groups[0]["lr"], "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay,
                 "amsgrad": False, "maximize": False, "foreach": None, "capturable": self.capturable, "differentiable": False,
                 "fused": None, "decoupled_weight_decay": True, "params": list(range(len(self.params)))}
        return {"state": state, "param_groups": [group]}

    def load_state_dict(self, sd):
        """torch.optim.AdamW's layout; the states keep this optimiser's number of bits"""
        groups = sd["param_groups"]
        order = [i for g in groups for i in g["params"]]
        if len(order) != len(self.params):
            raise ValueError(f"optimizer state covers {len(order)} parameters, the model has {len(self.params)}")
        g0 = groups[0]
        if g0.get("amsgrad", False) or g0.get("maximize", False):
            raise NotImplementedError("amsgrad / maximize optimizer states are not supported")
        plain = lambda v: tuple(v) if isinstance(v, (list, tuple)) else v  # noqa: E731
        differ = [k for k in ("lr", "betas", "eps", "weight_decay", "amsgrad", "maximize") if any(plain(g.get(k)) != plain(g0.get(k)) for g in groups)]
        if differ:
            raise ValueError(f"parameter groups with {', '.join(differ)} of their own: one group for all parameters is supported")
        values = {k: torch.zeros_like(v) for k, v in ops.adamw_state_values(self.state).items()}
        steps = set()
        for slot, p, o in zip(order, self.params, self.starts):
            st, n = sd["state"].get(slot), p.numel()
            if "master" in self.state:
                self.state["master"][o:o + n].copy_((st or {}).get("master_param", p.detach()).reshape(-1))
            if st is None:
                continue
            if tuple(st["exp_avg"].shape) != tuple(p.shape):
                raise ValueError(f"optimizer state {slot}: shape {tuple(st['exp_avg'].shape)} != parameter {tuple(p.shape)}")
            for k in values:
                values[k][o:o + n].copy_(st[k].reshape(-1))
            steps.add(int(float(st["step"])))
        if len(steps) > 1:
            raise ValueError(f"per-parameter AdamW step counts differ ({sorted(steps)}): one shared step is supported")
        ops.adamw_state_pack(self.state, values)
        self.step_count = steps.pop() if steps else 0
        self.param_groups[0]["lr"] = g0["lr"]
        self.sync_lr()
        self.betas, self.eps = tuple(g0.get("betas", self.betas)), g0.get("eps", self.eps)
        self.weight_decay = g0.get("weight_decay", self.weight_decay)


def _via_host(t):
    """gloo (CPU tests; several ranks on one GPU in the -m gpu tests) moves device tensors through the host"""
    import torch.distributed as dist
    return t.is_cuda and dist.get_backend() == "gloo"


def _broadcast(t, src):
    import torch.distributed as dist
    if _via_host(t):
        h = t.cpu()
        dist.broadcast(h, src)
        t.copy_(h)
    else:
        dist.broadcast(t, src)


def broadcast_replica(bucket, optim=None, src=0):
    """Make every rank an identical replica of rank `src` (start of training / after a resume): parameters, and the Adam
    moments + step when an optimizer is given.  nn.DataParallel re-broadcasts the parameters every step
    (hl_module:34-35); with one process per GPU once is enough, because every rank applies the same update."""
    import torch.distributed as dist
    if not (dist.is_available() and dist.is_initialized() and dist.get_world_size() > 1):
        return
    _broadcast(bucket.flat, src)
    bump_weight_epoch()
    if optim is not None:
        for t in optim.state_tensors():
            _broadcast(t, src)
        meta = torch.tensor([float(optim.step_count), float(optim.param_groups[0]["lr"])], device=bucket.flat.device,
                            dtype=torch.float64)
        _broadcast(meta, src)
        optim.step_count, optim.param_groups[0]["lr"] = int(meta[0].item()), float(meta[1].item())


FORCE_ALLREDUCE = False     # run the collective in a world of one as well (bench.py --init-dist, the RCCL smoke test)


def allreduce_grads(bucket, force=False):
    """One RCCL all-reduce (sum) of the whole gradient bucket (no-op without torch.distributed).  In a process group of ONE
    rank the collective is skipped unless `force` / FORCE_ALLREDUCE asks for it (RCCL then runs its kernel on the bucket --
    a sum over one rank -- in stream order between the backward and the optimiser: what tests/test_gpu_distributed.py checks)."""
    import torch.distributed as dist
    from . import ops
    ops.deferred_join()                      # reductions still on the library's side stream (normally joined at the end of backward)
    if dist.is_available() and dist.is_initialized() and (dist.get_world_size() > 1 or force or FORCE_ALLREDUCE):
        if _via_host(bucket.grad):
            h = bucket.grad.cpu()
            dist.all_reduce(h, op=dist.ReduceOp.SUM)
            bucket.grad.copy_(h)
        else:
            dist.all_reduce(bucket.grad, op=dist.ReduceOp.SUM)      # ONE RCCL all-reduce of the whole bucket
        return dist.get_world_size()
    return 1


def train_step(model, bucket, optim, inputs, target, neg_weight, grad_clip=None):
    """zero_grad -> forward -> SNRLP loss.mean() -> backward -> all-reduce -> clip -> Adam
    (tain_val.py:66-80 + hl_module:303-321,430-441).  Returns the (device) loss scalar."""
    from .functional import SnrlpLossFn
    from . import ops
    bucket.zero_grad()
    est = model(inputs)["output"]
    loss, _ = SnrlpLossFn.apply(est, target, neg_weight)
    ops.absmax_hints_clear()
    loss.backward()
    ops.deferred_join()                      # (the engine's final callback has done it: idempotent)
    ops.absmax_hints_clear()
    world = allreduce_grads(bucket)
    optim.step(grad_clip=grad_clip, world_size=world)
    return loss.detach()
