"""Leaf records held in 8 bits: quantised as they are written, scaled back as they are read.

The records of a trained tree are read far more often than written, and bound by memory when they
are.  A :class:`RecordCache` holds them in about a quarter of their size for serving: lookups by
point or by leaf id, and edits, with the calls of :class:`N3Tree`.  (The reference keeps records in
float32 and writes float16 to files, svox/svox.py:856.)
"""
import torch
from torch import nn

from . import csrc as _C
from .formats import DataFormat

__all__ = ["RecordCache"]

_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_VALUES = (torch.float32, torch.bfloat16, torch.float16)


class RecordCache(nn.Module):
    """The leaf records of ``tree`` (on a CUDA device) in 8 bits, as they are now.

    A record's colour values are codes of type ``dtype`` (``torch.int8`` or
    ``torch.float8_e4m3fn``) and one scale, a power of two, for every ``group`` neighbouring ones: by
    default a colour channel's coefficients, 32 values of a record without a colour basis.  The
    scale is the smallest that leaves the largest magnitude at most 127 after rounding (448 for
    e4m3), so a value is off by at most half a step of its code.  The last value, the density, is
    held as float16.  A group with a value that is not finite reads as NaN.

    The cache has its own copy of the tree's structure and does not follow later changes of the
    tree.  Writes and reads of one cache are to be ordered like those of a tensor.
    """

    def __init__(self, tree, dtype=torch.int8, group=None):
        super().__init__()
        if dtype not in _CODES:
            raise RuntimeError("dtype must be torch.int8 or torch.float8_e4m3fn")
        if not tree.data.is_cuda:
            raise RuntimeError("svox_b200 has no CPU records: move the tree to a CUDA device "
                               "(tree.cuda())")
        data = tree.data.detach()
        K = data.shape[-1]
        if group is None:
            fmt = tree.data_format
            basis = fmt.basis_dim if isinstance(fmt, DataFormat) and \
                fmt.format != DataFormat.RGBA else 0
            group = basis if basis > 0 else min(max(K - 1, 1), 32)
        self.data_dim, self.group, self.dtype = K, int(group), dtype
        self.data_format = tree.data_format
        size = _C.record_bytes(K, self.group)
        dev = data.device

        def copied(x, dtype):
            return x.detach().to(device=dev, dtype=dtype, copy=True).contiguous()

        self.register_buffer("child", copied(tree.child, torch.int32))
        self.register_buffer("offset", copied(tree.offset, torch.float32))
        self.register_buffer("invradius", copied(tree.invradius, torch.float32))
        n = self.child.numel()
        self.register_buffer("records", torch.zeros(n, size, dtype=torch.uint8, device=dev))
        self.register_buffer("_owner", torch.zeros(n, dtype=torch.int32, device=dev),
                             persistent=False)
        self._write(None, False, data.reshape(n, K), self.offset, self.invradius)

    def __len__(self):
        return self._buffers["records"].shape[0]

    def extra_repr(self):
        return (f"records={len(self)}, data_dim={self.data_dim}, dtype={self.dtype}, "
                f"group={self.group}")

    # What the bytes mean goes with them: a state of another kind of cache is refused, and a state is
    # taken whole or not at all.
    def get_extra_state(self):
        return {"data_dim": self.data_dim, "group": self.group, "dtype": str(self.dtype)}

    def set_extra_state(self, state):
        mine = self.get_extra_state()
        if state != mine:
            raise RuntimeError(f"the state is that of a record cache with {state}, this one has {mine}")

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                              unexpected_keys, error_msgs):
        # (buffers are copied before set_extra_state is called)
        try:
            self._check_state({k[len(prefix):]: v for k, v in state_dict.items()
                               if k.startswith(prefix)})
        except RuntimeError as error:
            error_msgs.append(str(error))
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys,
                                      unexpected_keys, error_msgs)

    def _check_state(self, state):
        names = ["child", "offset", "invradius", "records"]
        given = [name for name in (*names, "_extra_state") if name in state]
        if not given:
            return              # (the state of something else: for `strict` to judge)
        if len(given) <= len(names):
            raise RuntimeError(f"the state of a record cache has only {', '.join(given)}")
        self.set_extra_state(state["_extra_state"])
        for name in names:
            new, old = state[name], self._buffers[name]
            if new.shape != old.shape or new.dtype != old.dtype:
                raise RuntimeError(f"{name} of the state of a record cache is {tuple(new.shape)} "
                                   f"{new.dtype}, here {tuple(old.shape)} {old.dtype}")

    def _write(self, where, points, values, offset, scaling):
        b = self._buffers
        if values.requires_grad:
            if torch.is_grad_enabled():
                raise RuntimeError("a record cache takes no gradient: detach the values")
            values = values.detach()
        if values.dtype not in _VALUES:
            values = values.float()
        _C.host().records_write(b["records"], b["_owner"], b["child"], offset, scaling,
                                self.data_dim, self.group, _CODES[self.dtype], where, points,
                                values.contiguous())

    def _read(self, where, points, dtype, offset, scaling):
        b = self._buffers
        return _C.host().records_read(b["records"], b["child"], offset, scaling, self.data_dim,
                                      self.group, _CODES[self.dtype], where, points, dtype)

    def _frame(self, world):
        b = self._buffers
        if world:
            return b["offset"], b["invradius"]
        return torch.zeros_like(b["offset"]), torch.ones_like(b["invradius"])

    def set(self, points, values, world=True):
        """Quantise row q of ``values`` ``(Q, data_dim)`` into the record of the leaf that holds
        ``points[q]`` (as :meth:`N3Tree.set`; of several points in one leaf the last one counts)."""
        self._write(self._points(points), True, values, *self._frame(world))

    def forward(self, points, dtype=torch.float32, world=True):
        """Records ``(Q, data_dim)`` of the leaves that hold ``points`` ``(Q, 3)``, in ``dtype``
        (as :meth:`N3Tree.forward`; no gradient)."""
        return self._read(self._points(points), True, dtype, *self._frame(world))

    def write(self, ids, values):
        """Quantise row q of ``values`` into record ``ids[q]``: a packed leaf id as a query returns
        it, in any order; of several rows for one record the last one counts.  An id out of range is
        skipped and noticed by ``csrc.check_device_status()``."""
        self._write(ids.contiguous(), False, values, *self._frame(True))

    def read(self, ids=None, dtype=torch.float32):
        """Records of the packed leaf ids ``(Q,)`` (all records by default), in ``dtype``.  An id out
        of range reads as NaN and is noticed by ``csrc.check_device_status()``."""
        return self._read(None if ids is None else ids.contiguous(), False, dtype,
                          *self._frame(True))

    def _points(self, points):
        assert not points.requires_grad  # Grad wrt points not supported
        assert points.dim() == 2
        if points.dtype != torch.float32:
            points = points.to(torch.float32)
        return points.contiguous()
