"""Many owners' low-rank adapters on one frozen model: the weights of one projection's adapters (`AdapterBank`) and the description of which
rows belong to whom (`RequestPlan`), the two handles of `ops.adapter_linear`.

A watermark LoRA that has been baked for an owner (`inference.create_watermark_lora`) is an ordinary LoRA with matrices of its own.  Fusing it
into the weights serves one owner per model copy; `ops.lora_linear` shares one pair of matrices between all samples.  Here every request of a
batch names its adapter, and the batch still runs the shared projection as one product."""
import threading

import numpy as np
import torch
import torch.nn as nn
from torch.optim.optimizer import register_optimizer_step_post_hook

from . import _lib as L

MAX_RANK = 1024
MAX_ADAPTERS = 65535


def _count_fused_step(optimizer, args, kwargs):
    """torch's fused optimizers write parameters without raising their versions, by which a bank tells that its weights have changed."""
    for group in optimizer.param_groups:
        if group.get("fused"):
            for p in group["params"]:
                if getattr(p, "_aql_bank_weights", False) and p.grad is not None:
                    torch.autograd.graph.increment_version(p)


_fused_hook = None


class AdapterBank:
    """G adapters of one projection [N, K], stacked at one rank.

    ``down`` [G, r, K] and ``up`` [G, N, r] in bf16 or fp32; ``ranks[g]`` <= r says how much of adapter g is used (None: all of it), ``scales[g]``
    multiplies it (None: 1).  The kernels read bf16 copies laid out once.  ``trainable``: ``down`` / ``up`` become fp32 parameters, their
    gradients are fp32, and the copies follow after an optimizer step: `refresh` lays them out again when the parameters' versions
    have changed (ops.adapter_linear calls it; writes that raise no version -- through ``.data``, by collectives such as
    ``dist.broadcast``, by an optimizer step inside a captured graph -- need ``refresh(force=True)`` behind them).  A graph reads the stacks as they are at its replay: an eager step between replays needs `refresh` behind it;
    a call in a capture that finds them stale is refused, and ``refresh(force=True)`` in a capture is for the replays of that graph alone."""

    @torch.inference_mode(False)
    def __init__(self, down, up, ranks=None, scales=None, trainable=False, device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise L.AqlError("AdapterBank needs an MI355X (cuda device); there is no CPU path")
        if down.dim() != 3 or up.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2]:
            raise ValueError(f"AdapterBank: down [G, r, K] and up [G, N, r], not {tuple(down.shape)} and {tuple(up.shape)}")
        for t in (down, up):
            if t.dtype not in (torch.bfloat16, torch.float32):
                raise ValueError(f"AdapterBank: bfloat16 or float32 weights, not {t.dtype}")
        self.G, self.rank, self.K = down.shape
        self.N = up.shape[1]
        if not (1 <= self.G <= MAX_ADAPTERS and 1 <= self.rank <= MAX_RANK and self.K % 8 == 0 and self.N % 8 == 0 and self.K and self.N):
            raise ValueError(f"AdapterBank: 1 to {MAX_ADAPTERS} adapters of rank 1 to {MAX_RANK} on sides that are multiples of 8, "
                             f"not {self.G} of rank {self.rank} on [{self.N}, {self.K}]")
        self.ranks = [self.rank] * self.G if ranks is None else [int(r) for r in ranks]
        self.scales = [1.0] * self.G if scales is None else [float(s) for s in scales]
        if len(self.ranks) != self.G or len(self.scales) != self.G or not all(0 <= r <= self.rank for r in self.ranks):
            raise ValueError("AdapterBank: one rank of at most r and one scale for each adapter")
        self.R = (self.rank + 7) // 8 * 8    # the stacks' rank
        self.trainable, self.device = bool(trainable), dev
        h = self.handle = L.native().Bank()  # what the kernels' binding reads
        h.G, h.r, h.R, h.K, h.N, h.trainable = self.G, self.rank, self.R, self.K, self.N, self.trainable
        h.ranks = torch.tensor(self.ranks, dtype=torch.int32, device=dev)
        h.scales = torch.tensor(self.scales, dtype=torch.float32, device=dev)
        self._live = torch.arange(self.rank, device=dev)[None] < h.ranks[:, None]      # [G, r]
        h.a = torch.zeros(self.G, self.R, self.K, dtype=torch.bfloat16, device=dev)
        h.b = torch.zeros(self.G, self.N, self.R, dtype=torch.bfloat16, device=dev)
        self._transposed, self._lock = False, threading.Lock()
        if trainable:
            self.down = nn.Parameter(down.detach().to(device=dev, dtype=torch.float32, copy=True))
            self.up = nn.Parameter(up.detach().to(device=dev, dtype=torch.float32, copy=True))
            self.down._aql_bank_weights = self.up._aql_bank_weights = True
            global _fused_hook
            if _fused_hook is None:
                _fused_hook = register_optimizer_step_post_hook(_count_fused_step)
        else:
            # (a copy of an inference tensor: `refresh` goes by version counters)
            self.down, self.up = (t.detach().to(dev, copy=t.is_inference()) for t in (down, up))
        h.down, h.up = self.down, self.up
        self.refresh()
        if trainable:
            self.lay_out_transposed()

    def __reduce__(self):                    # copied and pickled by what it was made from (a U-Net that carries banks can be, too)
        return AdapterBank, (self.down.detach(), self.up.detach(), self.ranks, self.scales, self.trainable, str(self.device))

    @classmethod
    def from_layers(cls, layers, trainable=False, device="cuda"):
        """From LoRA layers (lora.LoRALinearLayer / LoRAConv2dLayer, 1x1) of one projection; ``network_alpha / rank`` becomes the scale."""
        ranks = [int(ly.rank) for ly in layers]
        r = max(ranks)
        downs, ups, scales = [], [], []
        for ly in layers:
            d = ly.down.weight.detach().reshape(ly.rank, -1).float()
            u = ly.up.weight.detach().reshape(-1, ly.rank).float()
            downs.append(nn.functional.pad(d, (0, 0, 0, r - ly.rank)))
            ups.append(nn.functional.pad(u, (0, r - ly.rank)))
            alpha = getattr(ly, "network_alpha", None)
            scales.append(1.0 if alpha is None else float(alpha) / ly.rank)
        return cls(torch.stack(downs), torch.stack(ups), ranks=ranks, scales=scales, trainable=trainable, device=device)

    def parameters(self):
        return [self.down, self.up] if self.trainable else []

    def refresh(self, force=False):
        h, r, live = self.handle, self.rank, self._live
        if h.fresh() and not force:
            return
        with self._lock:                     # of threads that come together the first lays out
            if h.fresh() and not force:
                return
            if not force and torch.cuda.is_current_stream_capturing():
                raise L.AqlError("AdapterBank: the weights have changed since they were laid out: call refresh() before the capture, or refresh(force=True) in it "
                                 "for a graph that lays them out at every replay")
            h.begin_layout()                 # behind what other threads and streams still read; backward passes of older calls are refused from here on
            with torch.no_grad():            # in place: a captured graph keeps reading these buffers
                h.a[:, :r].copy_(torch.where(live[:, :, None], self.down, torch.zeros((), dtype=self.down.dtype, device=self.device)))
                h.b[:, :, :r].copy_(torch.where(live[:, None, :], self.up, torch.zeros((), dtype=self.up.dtype, device=self.device)))
                if self._transposed:
                    h.at.copy_(h.a.transpose(1, 2))
                    h.bt.copy_(h.b.transpose(1, 2))
            h.end_layout()

    def lay_out_transposed(self):
        """B^T [G, R, N] and A^T [G, K, R], the stacks as the backward-data pass reads them: at once for a trainable bank, for others when an input
        first asks for a gradient."""
        if self._transposed:
            return
        if torch.cuda.is_current_stream_capturing():
            raise L.AqlError("AdapterBank: call lay_out_transposed() before capturing a pass that differentiates a frozen bank's input")
        with self._lock:                     # two threads may come here together: the first lays out
            if self._transposed:
                return
            h = self.handle
            h.reads()
            at, bt = h.a.transpose(1, 2).contiguous(), h.b.transpose(1, 2).contiguous()
            torch.cuda.current_stream(self.device).synchronize()      # once: later calls may come on other streams
            h.publish(at, bt)
            self._transposed = True


def banks_of(module):
    """The banks on the hosts inside ``module``."""
    return [m.adapter_bank for m in module.modules() if getattr(m, "adapter_bank", None) is not None]


class RequestPlan:
    """Which rows use which adapter: request i has ``lengths[i]`` rows (None: all requests have the same number, whatever the rows of the call) and
    adapter ``adapters[i]`` (-1: none).  Requests follow each other in the rows.  The tables are built on the host once and live on the device;
    one plan serves every projection of a model, and calls with any number of rows per request when ``lengths`` is None."""

    def __init__(self, adapters, lengths=None, device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise L.AqlError("RequestPlan needs an MI355X (cuda device); there is no CPU path")
        ids = np.asarray([int(a) for a in adapters], dtype=np.int64)
        if ids.size and (ids.min() < -1 or ids.max() >= MAX_ADAPTERS):
            raise ValueError(f"RequestPlan: adapters are numbered from 0 to {MAX_ADAPTERS - 1}; -1 is none")
        self.equal = lengths is None
        self.adapters, self.device = [int(a) for a in ids], dev
        self.lengths = None if self.equal else [int(x) for x in lengths]
        self.requests = int(ids.size)
        n = np.ones(ids.size, dtype=np.int64) if self.equal else np.asarray(self.lengths, dtype=np.int64)
        if n.size != ids.size or (n.size and n.min() < 0):
            raise ValueError("RequestPlan: one length of 0 or more for each request")
        if int(n.sum()) >= (1 << 31) - 256:
            raise ValueError("RequestPlan: too many rows")
        ids, n = ids[n > 0], n[n > 0]
        unit_rows = int(np.gcd.reduce(n)) if n.size else 1            # the tables count in the largest unit that divides all requests
        n = n // unit_rows
        self.units = int(n.sum())
        first = np.flatnonzero(np.r_[True, ids[1:] != ids[:-1]]) if ids.size else np.zeros(0, dtype=np.int64)
        begin = np.r_[0, np.cumsum(n)]
        start = np.r_[begin[first], self.units] if ids.size else np.zeros(1, dtype=np.int64)     # [n + 1], neighbours of one adapter joined
        seg = ids[first] if ids.size else ids
        self.max_id = int(seg.max()) if seg.size else -1
        size = np.diff(start)
        unit_id = np.repeat(seg, size)
        # sorted order of the rows that have an adapter, for the weight gradients
        perm = np.argsort(unit_id, kind="stable")[int((unit_id < 0).sum()):]
        used, count = np.unique(unit_id[perm], return_counts=True)
        used_pos = np.r_[0, np.cumsum(count)]
        slot = np.full(max(self.max_id + 1, 1), -1, dtype=np.int64)
        slot[used] = np.arange(used.size)
        parts = dict(unit_id=unit_id, perm=perm, used_pos=used_pos, slot=slot)
        flat = np.concatenate([p.astype(np.int32) for p in parts.values()])
        h = self.handle = L.native().Plan()  # what the kernels' binding reads
        self.table = h.table = torch.from_numpy(flat).to(dev)
        h.at = np.r_[0, np.cumsum([p.size for p in parts.values()])[:-1]].tolist()
        h.start = start.tolist()
        h.units, h.unit_rows, h.requests, h.live_units = self.units, unit_rows, self.requests, int(perm.size)
        h.equal, h.max_id = self.equal, self.max_id
        h.nseg = int(seg.size) if self.max_id >= 0 else 0              # no adapters at all: no segments
        h.nused, h.nslot = int(used.size), int(slot.size)

    def __reduce__(self):
        return RequestPlan, (self.adapters, self.lengths, str(self.device))
