"""Clip + SGD for the train step, one pass over device-resident tables instead of ~3000 small aten
launches: the reference's torch.nn.utils.clip_grad_norm(params, 5.0) followed by
torch.optim.SGD(momentum, weight decay on the non-'bn' group).step() (model.py:352-358, 441-444)."""
import ctypes as C

import numpy as np
import torch

from . import _lib

CHUNK = 1 << 16
CAPTURES = 16          # steps that can be captured after an eager one (their tables cannot be made inside of a capture)
_EAGER_FIRST = "take an eager step over the same parameters before captured ones (at least %d may follow it)" % (CAPTURES // 2)


class _Captured(list):
    """What captured steps over a weight hold, on the weight.  Copies and pickles of the weight start without."""

    def __reduce__(self):
        return _Captured, ()


class ClippedSGD(object):
    """param_groups like torch.optim.SGD's ([{'params': [...], 'weight_decay': w}, ...]).  step(max_norm)
    clips over every parameter that holds a gradient and applies momentum SGD; the total gradient norm
    is left in `last_norm` (0-d float32 device tensor, no host sync)."""

    def __init__(self, param_groups, lr, momentum=0.0):
        self.param_groups = []
        for g in param_groups:
            g = dict(g)
            g["params"] = list(g["params"])
            g.setdefault("weight_decay", 0.0)
            g.setdefault("lr", lr)
            g.setdefault("momentum", momentum)
            self.param_groups.append(g)
        self.state = {}                      # param -> momentum buffer
        self.skipped = None                  # device int32: steps skipped (non-finite gradient norm OR a clamp veto)
        self.skipped_clamped = None          # device int32: of those, the steps vetoed for clamped operand blocks
        self._plan_key, self._plan = None, None
        self._ring, self._turn = [], 0       # pinned staging buffers of the pointer tables
        self._spares, self._captured = [], []         # tables for captured steps; what those read and write
        self.capturing = False               # inside a HIP-graph capture: no event waits (the tables are static)
        self.last_norm = None

    def _hyper(self):
        """lr / momentum are read from the groups at step time, like torch.optim.SGD (an LR scheduler or
        `optimizer.param_groups[i]['lr'] = ...` takes effect); the fused kernel applies ONE pair to every
        tensor, so the groups must agree."""
        lrs = {float(g["lr"]) for g in self.param_groups if g["params"]}
        moms = {float(g["momentum"]) for g in self.param_groups if g["params"]}
        if len(lrs) > 1 or len(moms) > 1:
            raise ValueError("ClippedSGD applies one lr / momentum to all parameter groups (got lr %s, "
                             "momentum %s)" % (sorted(lrs), sorted(moms)))
        return (lrs.pop() if lrs else 0.0), (moms.pop() if moms else 0.0)

    @property
    def lr(self):
        return self._hyper()[0]

    @lr.setter
    def lr(self, value):
        for g in self.param_groups:
            g["lr"] = float(value)

    @property
    def momentum(self):
        return self._hyper()[1]

    def skipped_steps(self):
        """Steps whose update was skipped on the device because the gradient norm was inf / NaN (host sync)."""
        return (int(self.skipped.item()) if self.skipped is not None else 0) + getattr(self, "_skipped_loaded", 0)

    def skipped_clamped_steps(self):
        """Of skipped_steps(): the steps vetoed because an fp16 operand block had to clamp in them (host sync)."""
        return int(self.skipped_clamped.item()) if self.skipped_clamped is not None else 0

    def state_dict(self):
        """Momentum buffers by position in the flattened parameter groups + the groups' hyper-parameters
        (the layout of torch.optim.SGD.state_dict)."""
        flat = [p for g in self.param_groups for p in g["params"]]
        idx = {id(p): i for i, p in enumerate(flat)}
        groups, k = [], 0
        for g in self.param_groups:
            d = {key: v for key, v in g.items() if key != "params"}
            d["params"] = list(range(k, k + len(g["params"])))
            k += len(g["params"])
            groups.append(d)
        return {"state": {idx[id(p)]: {"momentum_buffer": b} for p, b in self.state.items() if id(p) in idx},
                "param_groups": groups, "skipped_steps": self.skipped_steps()}

    def load_state_dict(self, sd):
        flat = [p for g in self.param_groups for p in g["params"]]
        if len(sd["param_groups"]) != len(self.param_groups):
            raise ValueError("loaded state dict has a different number of parameter groups")
        for g, d in zip(self.param_groups, sd["param_groups"]):
            if len(d["params"]) != len(g["params"]):
                raise ValueError("loaded state dict contains a parameter group of a different size")
            g.update({key: v for key, v in d.items() if key != "params"})
        held = self._held()
        self.state = {}
        self._skipped_loaded = int(sd.get("skipped_steps", 0))     # (added to the device counter's value)
        with torch.no_grad():
            for i, st in sd["state"].items():
                p = flat[int(i)]
                b = st.get("momentum_buffer")
                if b is not None:
                    own = held.pop(id(p), (p, None))[1]            # (a captured step's is loaded in place: its replays go on from it)
                    own = torch.zeros_like(p, memory_format=torch.preserve_format) if own is None else own
                    self.state[p] = own.copy_(b)
            for p, own in held.values():
                self.state[p] = own.zero_()

    def zero_grad(self, set_to_none=True):
        for g in self.param_groups:
            for p in g["params"]:
                if set_to_none:
                    p.grad = None
                elif p.grad is not None:
                    p.grad.zero_()

    def replayed(self):
        """To be called when graphs that captured step() were replayed, before anything else reads the weights: what layers
        keep of a weight (its 16-bit parts, folded biases) goes by the weight's version counter, and a replay writes weights
        without moving it."""
        ps = list({id(p): p for c in self._captured for p in c[0]}.values())
        if ps:
            torch._C._autograd._unsafe_set_version_counter(ps, [p._version + 1 for p in ps])

    def _held(self):
        """id(weight) -> (weight, momentum buffer) of captured steps."""
        return {id(p): (p, b) for c in self._captured for p, b in zip(c[0], c[1])}

    def _active(self):
        out = []
        for g in self.param_groups:
            for p in g["params"]:
                if p.grad is not None:
                    out.append((p, float(g["weight_decay"])))
        return out

    def _chunks(self, numels, wds, device):
        key = (tuple(numels), tuple(wds))
        if key != self._plan_key:
            if self._capturing():
                raise RuntimeError(_EAGER_FIRST)
            ct, co = [], []
            for i, n in enumerate(numels):
                for off in range(0, n, CHUNK):
                    ct.append(i)
                    co.append(off)
            self._plan = (torch.tensor(ct, dtype=torch.int32, device=device),
                          torch.tensor(co, dtype=torch.int64, device=device),
                          torch.tensor(numels, dtype=torch.int64, device=device),
                          torch.empty(max(len(ct), 1), dtype=torch.float64, device=device),
                          torch.tensor(wds, dtype=torch.float32, device=device))
            self._plan_key = key
        return self._plan

    @torch.no_grad()
    def step(self, max_norm, veto=None):
        """veto: float32 [1] device tensor or None; > 0 = do not apply this step (conv_hip.clamp_veto(), or the
        all-reduced one of parallel.GradientAllReducer): the update is skipped on the device through the same guard
        as a non-finite gradient norm and counted in `skipped` and `skipped_clamped`; `last_norm` stays the real
        norm.  No host sync either way.

        Steps may be captured into graphs, after an eager step over the same parameters (eight or more in a row).  Replays use the
        hyper-parameters of the capture and the gradient tensors that were there: keep those, and call replayed()."""
        act = self._active()
        if not act:
            return None
        dev = act[0][0].device
        if dev.type != "cuda":
            raise RuntimeError("ClippedSGD runs on the GPU only (no CPU fallback in sln_amodal_amd)")
        ps, gs, bs = self._buffers(act)
        ct, co, numel, partial, wd = self._chunks([p.numel() for p in ps], [w for _, w in act], dev)
        tab = self._upload(ps, gs, bs, dev)[1]
        sq = torch.empty(1, dtype=torch.float64, device=dev)
        lr, momentum = self._hyper()
        st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        L = _lib.lib()
        vp = lambda t: C.c_void_p(t.data_ptr())
        nch = ct.numel() if sum(p.numel() for p in ps) else 0
        _lib.check(L.sln_grad_sqnorm_f32(vp(tab[1]), vp(numel), vp(ct), vp(co), nch, CHUNK, vp(partial), vp(sq),
                                         st), "sln_grad_sqnorm_f32")
        sq_guard = self._guard(sq, veto)
        _lib.check(L.sln_sgd_clip_step_f32(vp(tab[0]), vp(tab[1]), vp(tab[2]), vp(numel), vp(wd), vp(ct), vp(co),
                                           nch, CHUNK, vp(sq_guard), float(max_norm), lr, momentum, vp(self.skipped),
                                           st), "sln_sgd_clip_step_f32")
        # caches keyed by the weights' version counters (split weight parts) must see the update
        torch._C._autograd._unsafe_set_version_counter(ps, [p._version + 1 for p in ps])
        self._keep = (tab, gs, sq_guard)      # alive until the next step: the launches above are asynchronous
        self.last_norm = sq.sqrt().to(torch.float32)[0]
        return self.last_norm

    def _buffers(self, act):
        """Parameters, gradients (element i of the gradient is element i of the weight) and momentum buffers."""
        ps, gs, bs = [], [], []
        capturing = self._capturing()
        if self.skipped is None:
            if capturing:
                raise RuntimeError(_EAGER_FIRST)
            self.skipped, self.skipped_clamped = (torch.zeros(1, dtype=torch.int32, device=act[0][0].device) for _ in range(2))
        for p, _ in act:
            g = p.grad
            if p.dtype != torch.float32 or g.dtype != torch.float32:
                raise TypeError("%s needs float32 parameters and gradients" % type(self).__name__)
            if not (p.is_contiguous() or (p.dim() == 4 and p.is_contiguous(memory_format=torch.channels_last))):
                raise ValueError("parameters must be dense")
            if g.stride() != p.stride():       # element i of the gradient must be element i of the weight
                g = torch.empty_like(p).copy_(g)
            b = self.state.get(p)
            if b is None:
                if capturing:                  # (its clearing would be part of every replay)
                    raise RuntimeError(_EAGER_FIRST)
                b = self.state[p] = torch.zeros_like(p, memory_format=torch.preserve_format)
            elif b.stride() != p.stride():     # (and of the momentum: the weight may have changed its memory format)
                if capturing or id(p) in self._held():
                    raise RuntimeError("a weight of a captured step cannot change its memory format")
                b = self.state[p] = torch.empty_like(p).copy_(b)
            ps.append(p); gs.append(g); bs.append(b)
        return ps, gs, bs

    def _capturing(self):
        return self.capturing or torch.cuda.is_current_stream_capturing()

    def _upload(self, ps, gs, bs, dev):
        """Pointer tables [3, n] (weights, gradients, momentum), as lists and on the device: gradients are fresh
        allocations every step, so the tables are re-sent each time -- from pinned staging buffers and asynchronously, so
        the host never waits for the GPU here (a pageable copy would drain the stream once per step).  A staging buffer
        is reused only after the copy that read it has completed (4 in flight); one that a captured graph copies from is
        never written again (its replays read it)."""
        n = len(ps)
        capturing = self._capturing()
        if capturing:
            if not torch.cuda.is_current_stream_capturing():
                raise RuntimeError("`capturing` is set, but nothing is being captured on this stream")
            if not self._spares or self._spares[0].shape[1] != n:
                raise RuntimeError(_EAGER_FIRST)
            stage = [self._spares.pop(), None]
            # everything of the optimiser's own that the replays touch lives as long as the optimiser or one of the weights,
            # whatever later eager steps put in its place: tables, chunk plan, momentum, and the memory that the weights had
            step = (ps, bs, stage[0], self._plan, [p.detach() for p in ps], self.skipped, self.skipped_clamped)
            self._captured.append(step)
            for p in ps:                       # (its replays write p without moving p's version: nothing made from p is kept)
                if not getattr(p, "_sln_captured", None):
                    p._sln_captured = _Captured()
                p._sln_captured.append(step)
        else:
            if not self._ring or self._ring[0][0].shape[1] != n:
                self._ring = [[torch.empty((3, n), dtype=torch.int64, pin_memory=True), None] for _ in range(4)]
            if len(self._spares) < CAPTURES // 2 or self._spares[0].shape[1] != n:
                self._spares = list(torch.empty((CAPTURES, 3, n), dtype=torch.int64, pin_memory=True))
            stage = self._ring[self._turn % len(self._ring)]
            self._turn += 1
            if stage[1] is not None:
                stage[1].synchronize()
        host = [[t.data_ptr() for t in ts] for ts in (ps, gs, bs)]
        stage[0].numpy()[:] = host
        tab = torch.empty((3, n), dtype=torch.int64, device=dev)
        tab.copy_(stage[0], non_blocking=True)
        if not capturing:
            stage[1] = torch.cuda.Event()
            stage[1].record()
        return host, tab

    def _guard(self, sq, veto):
        """The guard's input: +inf instead of the squared norm when the step is vetoed (two 5-us elementwise ops)."""
        if veto is None:
            return sq
        hit = veto.reshape(1) > 0
        # (a step that is non-finite anyway is counted as that, not as clamped)
        self.skipped_clamped += (hit & torch.isfinite(sq)).to(torch.int32)
        return torch.where(hit, torch.full_like(sq, float("inf")), sq)


class _MuonDesc(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("momentum", C.c_void_p), ("rows", C.c_int32),
                ("cols", C.c_int32), ("lr", C.c_float), ("decay", C.c_float)]


class ClippedMuon(ClippedSGD):
    """Clip + orthogonalised momentum for the weight matrices, ClippedSGD's rule for everything else, in one step over
    all tensors (csrc/ortho.hip).  A group with "orthogonal": True holds parameters of two or more axes, each read as
    the matrix [first axis][all the others] (in memory order: a permutation of the columns permutes the result's); with
    g clipped by the global norm over ALL parameters,

        b <- momentum b + g;  u = g + momentum b (nesterov) or b
        p <- p (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) orthogonalize(u, steps, eps)

    Orthogonal groups have an lr, momentum, weight_decay of their own (one momentum for all of them); the other groups
    agree on one lr and momentum, like ClippedSGD's; setting `lr` sets theirs and scales the orthogonal ones'.  The same
    guard: a step with a non-finite gradient norm or a veto writes nothing and is counted.  Hyper-parameters are read when
    step() is called; a captured step keeps them."""

    def __init__(self, param_groups, lr, momentum=0.95, nesterov=True, steps=5, eps=1e-7):
        super(ClippedMuon, self).__init__(param_groups, lr, momentum)
        self.nesterov, self.steps, self.eps = bool(nesterov), int(steps), float(eps)
        if not 1 <= self.steps <= 64 or not self.eps >= 1e-30:
            raise ValueError("ClippedMuon: 1 <= steps <= 64 and eps >= 1e-30 (got %r, %r)" % (steps, eps))
        seen = set()
        for g in self.param_groups:
            g["orthogonal"] = bool(g.get("orthogonal", False))
            for p in g["params"]:
                if id(p) in seen:
                    raise ValueError("a parameter appears twice in the parameter groups")
                seen.add(id(p))
                rows = p.shape[0] if p.dim() else 0
                cols = p.numel() // rows if rows else 0
                if g["orthogonal"] and (p.dim() < 2 or min(rows, cols) > 65535 or max(rows, cols) > 1 << 22):
                    raise ValueError("an orthogonal group takes matrices (two or more axes, at most 65535 x 2^22), got %s" %
                                     (tuple(p.shape),))

    def _split(self):
        rest = [g for g in self.param_groups if not g["orthogonal"]]
        return rest, [g for g in self.param_groups if g["orthogonal"]]

    def _hyper(self):
        """lr / momentum of the groups that are not orthogonal (of the orthogonal ones where there are no others)."""
        rest, ortho = self._split()
        groups = [g for g in (rest if any(g["params"] for g in rest) else ortho) if g["params"]]
        lrs, moms = {float(g["lr"]) for g in groups}, {float(g["momentum"]) for g in groups}
        if rest and any(g["params"] for g in rest) and (len(lrs) > 1 or len(moms) > 1):
            raise ValueError("ClippedMuon applies one lr / momentum to its non-orthogonal groups (got lr %s, "
                             "momentum %s)" % (sorted(lrs), sorted(moms)))
        return (min(lrs) if lrs else 0.0), (min(moms) if moms else 0.0)

    @property
    def lr(self):
        return self._hyper()[0]

    @lr.setter
    def lr(self, value):
        """The rate that the getter reads; the orthogonal groups' rates keep their ratio to it.  (Where it is zero, the ratio
        that they had when it was set to that.)"""
        rest, ortho = self._split()
        live = [float(g["lr"]) for g in (rest if any(g["params"] for g in rest) else ortho) if g["params"]]
        value, old = float(value), min(live, default=0.0)
        ratios = [g["lr"] / old if old else g.get("lr_ratio") for g in ortho]
        if None in ratios:
            raise ValueError("lr is 0: the ratio of the orthogonal groups' rates to it is not known, set them in param_groups")
        for g in rest:
            g["lr"] = value
        for g, ratio in zip(ortho, ratios):
            g["lr"] = value if ratio == 1.0 else value * ratio
            g["lr_ratio"] = ratio

    def load_state_dict(self, sd):
        if len(sd["param_groups"]) == len(self.param_groups):
            for g, d in zip(self.param_groups, sd["param_groups"]):
                if bool(d.get("orthogonal", g["orthogonal"])) != g["orthogonal"]:
                    raise ValueError("loaded state dict marks other parameter groups as orthogonal")
        super(ClippedMuon, self).load_state_dict(sd)

    @torch.no_grad()
    def step(self, max_norm, veto=None):
        """See ClippedSGD.step: the same arguments, guard and counters."""
        rest, mats, moms = [], [], set()
        for g in self.param_groups:
            if g["orthogonal"]:
                lr, decay = float(g["lr"]), 1.0 - float(g["lr"]) * float(g["weight_decay"])
                live = [(p, (lr, decay)) for p in g["params"] if p.grad is not None]
                mats += live
                if live:
                    moms.add(float(g["momentum"]))
            else:
                wd = float(g["weight_decay"])
                rest += [(p, wd) for p in g["params"] if p.grad is not None]
        act = rest + mats
        if not act:
            return None
        if len(moms) > 1:
            raise ValueError("ClippedMuon applies one momentum to its orthogonal groups (got %s)" % sorted(moms))
        dev = act[0][0].device
        if dev.type != "cuda":
            raise RuntimeError("ClippedMuon runs on the GPU only (no CPU fallback in sln_amodal_amd)")
        for p, _ in act:
            if p.device != dev or p.grad.device != dev:
                raise ValueError("ClippedMuon: the parameters and gradients of one step share a device")
        lr, momentum = self._hyper()
        with _lib.on_device(dev):
            ps, gs, bs = self._buffers(act)
            sizes = [p.numel() for p in ps]
            ct, co, numel, partial, wd = self._chunks(sizes, [w for _, w in rest] + [0.0] * len(mats), dev)
            host, tab = self._upload(ps, gs, bs, dev)
            row = 8 * len(ps)
            at = tab.data_ptr()
            sq = torch.empty(1, dtype=torch.float64, device=dev)
            st = _lib.stream_of(dev)
            L = _lib.lib()
            # (the workspace before the first launch: nothing is written if there is no memory for it)
            flat = []
            for i, (p, (glr, decay)) in enumerate(mats, len(rest)):
                rows = p.shape[0]
                cols = sizes[i] // rows if rows else 0
                flat.append((host[0][i], host[1][i], host[2][i], rows, cols,
                             glr * max(1.0, rows / cols) ** 0.5 if cols else 0.0, decay))
            flat.sort(key=lambda d: -min(d[3], d[4]))            # (the longest products first: the launches end together)
            descs = (_MuonDesc * len(flat))(*flat)
            nbytes = L.sln_muon_step_workspace_bytes(descs, len(flat))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
            nch = ct.numel() if sum(sizes) else 0
            num, ctp, cop = numel.data_ptr(), ct.data_ptr(), co.data_ptr()
            _lib.check(L.sln_grad_sqnorm_f32(at + row, num, ctp, cop, nch, CHUNK, partial.data_ptr(), sq.data_ptr(), st),
                       "sln_grad_sqnorm_f32")
            guard = self._guard(sq, veto)
            # the vectors come first in the tables: their chunks are a prefix of the chunk list.  (The SGD kernel also
            # counts a skipped step; without vectors that is done here.)
            nrest = sum(-(-n // CHUNK) for n in sizes[:len(rest)])
            if nrest:
                _lib.check(L.sln_sgd_clip_step_f32(at, at + row, at + 2 * row, num, wd.data_ptr(), ctp, cop, nrest, CHUNK,
                                                   guard.data_ptr(), float(max_norm), lr, momentum, self.skipped.data_ptr(),
                                                   st), "sln_sgd_clip_step_f32")
            else:
                self.skipped += (~torch.isfinite(guard)).to(torch.int32)
            if mats:
                _lib.check(L.sln_muon_step_f32(descs, len(flat), self.steps, self.eps, guard.data_ptr(), float(max_norm),
                                               moms.pop(), self.nesterov, ws.data_ptr() if nbytes else 0, nbytes, st),
                           "sln_muon_step_f32")
            torch._C._autograd._unsafe_set_version_counter(ps, [p._version + 1 for p in ps])
            self._keep = (tab, gs, guard)
            self.last_norm = sq.sqrt().to(torch.float32)[0]
        return self.last_norm
