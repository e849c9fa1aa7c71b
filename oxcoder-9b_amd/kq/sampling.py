"""The greedy pick of several requests' next tokens under penalties, biases and a grammar mask.

``Engine.head`` picks for one request from its bare logits (engine.py:323-331); ``Picker.pick`` takes the
logits of a batch and applies what a serving program is asked for on the way, in one launch (kq_logits_penalize).
"""
import torch

from . import _lib, ops


class Picker:
    """``pick`` for up to ``rows`` requests; holds the workspace and the picked ids.  Calls on one Picker share
    them and so must be ordered: one stream, or synchronised."""

    def __init__(self, rows, device="cuda"):
        n = ops.logits_workspace_bytes(rows)
        if not n:
            raise ValueError("rows must be 1..65535")
        buf = torch.zeros(n + 256, dtype=torch.uint8, device=device)
        self.ws = buf[-buf.data_ptr() % 256:][:n]
        self.rows = rows
        self.picked = torch.empty(rows, dtype=torch.int32, device=device)
        # what every call passes on, as addresses: the tensors stay as long as the picker
        self._held, self._keep = (self.picked.data_ptr(), self.ws.data_ptr(), n), (self.picked, buf)
        self._device, self._calls = self.ws.device, _lib.calls()

    def pick(self, logits, history=None, length=None, prompt=None, repetition=None, frequency=None, presence=None,
             bias_ids=None, bias_values=None, allowed=None, out=None):
        """The id of the largest logit of each row of ``logits`` [B][V] after the steps below (the smallest id among
        equal ones, -1 where the mask or the logits leave nothing above -1e30); int32 [B], valid until the next call.

        history: int32 [B][L] token ids of which the first length[b] count, the first prompt[b] of these from the
        prompt (default none); repetition, frequency, presence: float [B].  An id in the history: y / repetition where
        y > 0, else y * repetition; one that occurs c > 0 times after the prompt: y - frequency * c - presence.
        bias_ids int32 [B][n] and bias_values [B][n]: added (an id's last entry counts; an id below 0 is none).
        allowed: int32 [B or 1][ceil(V / 32)], bit id % 32 of word id / 32; other ids become -inf.
        out: [B][V] receives the logits after these steps (may be ``logits``)."""
        if logits.dim() == 1:
            logits = logits.unsqueeze(0)
            out = out.unsqueeze(0) if out is not None and out.dim() == 1 else out
        rows = logits.shape[0]
        if rows > self.rows:
            raise ValueError("%d rows, the picker holds %d" % (rows, self.rows))
        if logits.device != self._device:
            raise ValueError("logits must be a device tensor, on the picker's device")
        rc = self._calls.pick(*self._held, ops._stream(self._device) if logits.is_cuda else None, logits, history, length, prompt,
                              repetition, frequency, presence, bias_ids, bias_values, allowed, out)
        picked = self.picked if rows == self.rows else self.picked[:rows]
        if rc is None:                       # a tensor is not as it should be
            ops.logits_penalize(logits, history, length, prompt, repetition, frequency, presence, bias_ids, bias_values,
                                allowed, out, picked, self.ws)
        elif rc:
            _lib.check(rc)
        return picked
