"""Long-running streams on the ring-buffer step, with checkpoint / restore.

``StreamingRing`` keeps everything a stream needs on the device -- the last
K+1 observations (values, masks, times), the ring head and the SSM state --
and advances all streams by one event per ``step`` through
``streaming_interp_then_ssm`` (``streaming_inference_kernel.py:74-156``).
``checkpoint`` copies that state to host memory, ``restore`` puts it back, so
a service can persist its streams and resume them bit for bit.
"""
import torch

from .delta import gated_delta_rule, gated_delta_step
from .norm import group_norm_act
from .ops import streaming_interp_then_ssm

__all__ = ["StreamingRing", "DeltaStream"]

_STATE = ("ring_V", "ring_M", "ring_tau", "ring_head", "h")
_PARAMS = ("Abar", "Bbar", "D")


class StreamingRing:
    """Bt independent streams of H features with a (K+1)-slot observation ring.

    Abar, Bbar, D [H] f32 are the (shared) step parameters.  ``block_h`` is the
    feature-tile width over which mask sums decide "observed"; it is part of
    the stream's definition and is kept in checkpoints.
    """

    def __init__(self, Bt, H, K, Abar, Bbar, D, device=None, block_h=128, h0=None):
        device = torch.device(device) if device is not None else Abar.device
        if device.type != "cuda":
            raise ValueError("StreamingRing lives on a CUDA device (no CPU fallback)")
        if K < 0 or K + 1 > 64:
            raise ValueError("StreamingRing: K must be in [0, 63]")
        f32 = dict(device=device, dtype=torch.float32)
        self.K, self.block_h = int(K), int(block_h)
        self.Abar, self.Bbar, self.D = (t.to(**f32).contiguous() for t in (Abar, Bbar, D))
        self.ring_V = torch.zeros(Bt, K + 1, H, **f32)
        self.ring_M = torch.zeros(Bt, K + 1, H, **f32)
        self.ring_tau = torch.zeros(Bt, K + 1, **f32)
        self.ring_head = torch.zeros(Bt, device=device, dtype=torch.int32)
        self.h = torch.zeros(Bt, H, **f32) if h0 is None else h0.to(**f32).clone().contiguous()
        self.steps = 0

    @property
    def shape(self):
        return tuple(self.h.shape)

    def step(self, v_new, m_new, tau_new, C, y=None):
        """Ingest one event per stream (v_new, m_new, C [Bt,H]; tau_new [Bt]) and
        return y [Bt,H]; the ring, head and state advance in place."""
        y = streaming_interp_then_ssm(self.ring_V, self.ring_M, self.ring_tau, self.ring_head, v_new, m_new,
                                      tau_new, self.h, self.Abar, self.Bbar, C, self.D, y=y, BLOCK_H=self.block_h)
        self.steps += 1
        return y

    def checkpoint(self, pin_memory=False):
        """A host copy of the streams' state and parameters (a dict of CPU tensors
        and ints); the copy is complete when this returns."""
        ck = {"K": self.K, "block_h": self.block_h, "steps": self.steps}
        for name in _STATE + _PARAMS:
            t = getattr(self, name)
            host = torch.empty(t.shape, dtype=t.dtype, pin_memory=pin_memory)
            host.copy_(t, non_blocking=pin_memory)
            ck[name] = host
        torch.cuda.current_stream(self.h.device).synchronize()
        return ck

    def restore(self, ck):
        """Put a checkpoint taken from a ring of the same shape back in place."""
        if int(ck["K"]) != self.K or int(ck["block_h"]) != self.block_h:
            raise ValueError("StreamingRing.restore: checkpoint has K=%s block_h=%s, ring has K=%d block_h=%d"
                             % (ck["K"], ck["block_h"], self.K, self.block_h))
        for name in _STATE + _PARAMS:
            dst = getattr(self, name)
            src = ck[name]
            if tuple(src.shape) != tuple(dst.shape) or src.dtype != dst.dtype:
                raise ValueError("StreamingRing.restore: %s has shape %s/%s, expected %s/%s"
                                 % (name, tuple(src.shape), src.dtype, tuple(dst.shape), dst.dtype))
            dst.copy_(src)
        self.steps = int(ck["steps"])

    def save(self, path):
        torch.save(self.checkpoint(), path)

    @classmethod
    def load(cls, path, device="cuda"):
        ck = torch.load(path, map_location="cpu", weights_only=True)
        Bt, KR, H = ck["ring_V"].shape
        ring = cls(Bt, H, KR - 1, ck["Abar"], ck["Bbar"], ck["D"], device=device, block_h=ck["block_h"])
        ring.restore(ck)
        return ring


class DeltaStream:
    """S independent streams of a gated-delta-rule layer: the state h [S,H,P,N]
    f32 stays in place on the device, ``prefill`` advances every stream by a prompt,
    ``step`` by one token.  Outputs are normalised per token and head (group
    norm with H groups), then ``act``.  N at most 128 (256 for streams that only
    step).

    A_log [H]; weight, bias [H*P] (default 1 and 0), f32; scale defaults to
    N ** -0.5.
    """

    _TENSORS = ("A_log", "weight", "bias", "h")

    def __init__(self, S, H, P, N, A_log, weight=None, bias=None, scale=None, eps=1e-5, act="silu", device=None,
                 h0=None):
        device = torch.device(device) if device is not None else A_log.device
        if device.type != "cuda":
            raise ValueError("DeltaStream lives on a CUDA device (no CPU fallback)")
        if tuple(A_log.shape) != (H,):
            raise ValueError("DeltaStream: A_log must be [H]")
        if act not in ("silu", "none"):
            raise ValueError("DeltaStream: act must be 'silu' or 'none' (got %r)" % (act,))
        f32 = dict(device=device, dtype=torch.float32)
        self.A_log = A_log.to(**f32).contiguous()
        self.weight = torch.ones(H * P, **f32) if weight is None else weight.to(**f32).contiguous()
        self.bias = torch.zeros(H * P, **f32) if bias is None else bias.to(**f32).contiguous()
        self.scale = float(N) ** -0.5 if scale is None else float(scale)
        self.eps, self.act, self.tokens = float(eps), act, 0
        self.h = torch.zeros(S, H, P, N, **f32)
        if h0 is not None:
            if tuple(h0.shape) != (S, H, P, N):
                raise ValueError("DeltaStream: h0 must be [S,H,P,N]")
            self.h.copy_(h0)

    def _norm(self, y):
        H = self.h.shape[1]
        return group_norm_act(y.reshape(-1, y.shape[-1]), self.weight, self.bias, H, eps=self.eps,
                              act=self.act).view(y.shape)

    def prefill(self, u, B, C, dt, beta):
        """L tokens of every stream: u [S,L,H*P], B, C [S,L,G,N], dt, beta [S,L,H]; streams that
        are shorter are padded at their end with zeros (dt = beta = 0).  Returns [S,L,H*P]."""
        if u.dim() != 3 or u.shape[0] != self.h.shape[0]:
            raise ValueError("DeltaStream.prefill: u must be [S,L,H*P] with S = %d streams" % self.h.shape[0])
        y, _ = gated_delta_rule(u, self.A_log, B, C, dt, beta, scale=self.scale, h0=self.h, return_state=True,
                                h_last=self.h)
        self.tokens += u.shape[1]
        return self._norm(y)

    def step(self, x, B, C, dt, beta):
        """One token of every stream: x [S,H*P], B, C [S,G,N], dt, beta [S,H].  Returns [S,H*P]."""
        S, H, P, _ = self.h.shape
        if tuple(x.shape) != (S, H * P):
            raise ValueError("DeltaStream.step: x must be [S,H*P] = [%d,%d]" % (S, H * P))
        y = gated_delta_step(x.reshape(S, H, P), dt, self.h, self.A_log, B, C, beta, scale=self.scale)
        self.tokens += 1
        return self._norm(y.view(S, H * P))

    def checkpoint(self):
        """A host copy of the streams' state and parameters, complete when this returns."""
        ck = {"scale": self.scale, "eps": self.eps, "act": self.act, "tokens": self.tokens}
        ck.update((k, getattr(self, k).cpu()) for k in self._TENSORS)
        return ck

    def restore(self, ck):
        """Put a checkpoint of streams of the same shape back in place."""
        for k in self._TENSORS:
            if tuple(ck[k].shape) != tuple(getattr(self, k).shape):
                raise ValueError("DeltaStream.restore: %s has shape %s, expected %s"
                                 % (k, tuple(ck[k].shape), tuple(getattr(self, k).shape)))
        for k in self._TENSORS:
            getattr(self, k).copy_(ck[k])
        self.scale, self.eps, self.act, self.tokens = (float(ck["scale"]), float(ck["eps"]), str(ck["act"]),
                                                       int(ck["tokens"]))

    def save(self, path):
        torch.save(self.checkpoint(), path)

    @classmethod
    def load(cls, path, device="cuda"):
        ck = torch.load(path, map_location="cpu", weights_only=True)
        S, H, P, N = ck["h"].shape
        st = cls(S, H, P, N, ck["A_log"], device=device)
        st.restore(ck)
        return st
