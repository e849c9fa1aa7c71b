"""The greedy pick of several requests' next tokens under penalties, biases and a grammar mask, and the verification of
drafted tokens.

``Engine.head`` picks for one request from its bare logits (engine.py:323-331); ``Picker.pick`` takes the
logits of a batch and applies what a serving program is asked for on the way, in one launch (kq_logits_penalize).  ``Verifier.verify`` takes the
logits after a tree of drafted tokens and says which the target's probabilities accept (kq_verify).
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


class Verifier:
    """``verify`` for up to ``requests`` trees of up to ``nodes`` nodes over ``vocab`` ids; holds the workspace and the results.
    Calls on one Verifier share them and so must be ordered: one stream, or synchronised."""

    def __init__(self, requests, nodes, vocab, device="cuda"):
        n = ops.verify_workspace_bytes(requests, nodes, vocab)
        if not n:
            raise ValueError("%d requests of 1..%d nodes (65535 in all) over %d ids: not supported"
                             % (requests, _lib.KQ_MAX_TREE, vocab))
        buf = torch.empty(n + 256, dtype=torch.uint8, device=device)
        self.ws = buf[-buf.data_ptr() % 256:][:n]
        self.requests, self.nodes, self.vocab = requests, nodes, vocab
        self.accepted, self.token = (torch.empty(requests, dtype=torch.int32, device=device) for _ in range(2))
        self.path = torch.empty((requests, nodes), dtype=torch.int32, device=device)
        # what every call passes on, as addresses: the tensors stay as long as the verifier
        self._held = (self.accepted.data_ptr(), self.path.data_ptr(), self.token.data_ptr(), self.ws.data_ptr(), n)
        self._keep, self._device = (self.accepted, self.path, self.token, buf), self.ws.device
        self._calls = _lib.calls()

    def verify(self, logits, tokens, parents, uniform, temperature=None, draft=None):
        """(accepted, path, token), int32, valid until the next call: accepted[b] drafts of request b's tree are taken, path[b]
        lists their nodes from the root (node 0) on, then -1, and token[b] follows them (-1: no logit above -inf).

        logits [B * T][V]: row b * T + t follows node t of request b; tokens int32 [B][T] the nodes' ids; parents int32
        [B or 1][T], node 0's being -1 (another value: the request sits out, accepted and token -1); uniform float [B][T]
        random numbers in [0, 1): one for each node's test, node 0's for the token; temperature float [B] (default 1;
        0: greedy).  draft: [B * T][V] probabilities that node t's children were drawn from, each by itself; default: the
        drafts were not drawn (a drafter's likeliest tokens).  A token's chance is the target's own, whatever was drafted."""
        if not isinstance(logits, torch.Tensor) or logits.device != self._device:
            raise ValueError("logits must be a device tensor, on the verifier's device")
        if not isinstance(tokens, torch.Tensor) or tokens.dim() != 2 or logits.dim() != 2:
            raise ValueError("tokens must be [requests][nodes], logits [requests * nodes][vocabulary]")
        (B, T), V = tokens.shape, logits.shape[1]
        if B > self.requests or T > self.nodes or V > self.vocab:
            raise ValueError("%d requests of %d nodes over %d ids, the verifier holds %d of %d over %d"
                             % (B, T, V, self.requests, self.nodes, self.vocab))
        accepted, path, token = self.accepted, self.path, self.token
        if (B, T) != (self.requests, self.nodes):
            accepted, path, token = accepted[:B], path.view(-1)[:B * T].view(B, T), token[:B]
        rc = self._calls.verify(*self._held, ops._stream(self._device) if logits.is_cuda else None, logits, tokens, parents, uniform,
                                temperature, draft)
        if rc is None:                       # a tensor is not as it should be
            ops.verify(logits, tokens, parents, uniform, temperature, draft, accepted, path, token, self.ws)
        elif rc:
            _lib.check(rc)
        return accepted, path, token
