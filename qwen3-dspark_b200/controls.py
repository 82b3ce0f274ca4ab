"""Logits controls: penalties for repeated tokens, biases and grammar masks.

``TokenControls`` keeps, per request slot, the tables the kernels read (how often each
token was emitted, which tokens the prompt holds, the penalties and the biases) on the
GPU. ``control_logits`` applies them to the logits of a verify round or decode step,
``control_argmax`` returns each row's controlled maximum without writing the logits, and
``TokenControls.commit`` adds a round's emitted tokens, from device tensors, so a decode
loop never reads them back. The rows of a verified chunk see the chunk's own proposals:
row j counts proposals 1 .. j on top of the table.

The arithmetic (float32, one rounding per step; ``dspark_control_logits``):
seen tokens (in the prompt, or emitted) are divided (positive) or multiplied by
``repetition``; emitted ones lose ``frequency * count + presence``; the sum of a token's
biases (added up in list order) is added; tokens the row's mask forbids become ``mask_value``.
"""
import math

import torch

from . import _lib
from .kernels import _DTYPES, _on_device, _stream
from .kv_store import _upload


class TokenControls:
    """Control tables of ``slots`` requests over a vocabulary of ``vocab`` tokens.

    ``counts`` int16 [slots, vocab rounded up to 8] (saturating at 32767), ``prompt_bits``
    int32 [slots, words] (bit ``v & 31`` of word ``v >> 5``), ``penalties`` float32
    [slots, 3], ``bias_ids`` / ``bias_values`` [slots, max_bias] and ``bias_len`` [slots].
    All work is on the current stream of the tables' device.
    """

    def __init__(self, slots, vocab, *, device='cuda', max_bias=0):
        if any(type(x) is not int for x in (slots, vocab, max_bias)) or slots < 1 or vocab < 1 or max_bias < 0:
            raise ValueError('Positive slots and vocab and a nonnegative max_bias required')
        self.device = torch.device(device)
        if self.device.type != 'cuda':
            raise RuntimeError('Logits controls require a CUDA device; no CPU fallback')
        if self.device.index is None:
            self.device = torch.device('cuda', torch.cuda.current_device())
        self.slots, self.vocab, self.max_bias = slots, vocab, max_bias
        self.words = (vocab + 31) // 32
        dev = dict(device=self.device)
        self.counts = torch.zeros((slots, (vocab + 7) // 8 * 8), dtype=torch.int16, **dev)
        self.prompt_bits = torch.zeros((slots, self.words), dtype=torch.int32, **dev)
        self.penalties = torch.zeros((slots, 3), dtype=torch.float32, **dev)
        self.penalties[:, 0] = 1.0
        self.bias_ids = torch.zeros((slots, max_bias), dtype=torch.int32, **dev)
        self.bias_values = torch.zeros((slots, max_bias), dtype=torch.float32, **dev)
        self.bias_len = torch.zeros(slots, dtype=torch.int32, **dev)
        # the tables stay where they are: the kernels' arguments that name them
        self._table_args = (self.counts.data_ptr(), self.counts.stride(0), self.prompt_bits.data_ptr(),
                            self.prompt_bits.stride(0), self.penalties.data_ptr(), slots,
                            self.bias_ids.data_ptr() if max_bias else None,
                            self.bias_values.data_ptr() if max_bias else None, self.bias_len.data_ptr(), max_bias)
        self._slots = {}
        self._free = list(range(slots))

    # -- request lifecycle -----------------------------------------------------------
    def _ids(self, tokens, what):
        if tokens is None:
            return torch.empty(0, dtype=torch.long, device=self.device)
        if not isinstance(tokens, torch.Tensor):
            tokens = torch.tensor(list(tokens), dtype=torch.long)
        if tokens.ndim != 1 or tokens.dtype not in (torch.long, torch.int32):
            raise ValueError(f'{what} must be one-dimensional integer token ids')
        if not tokens.is_cuda and tokens.numel() and not 0 <= int(tokens.min()) <= int(tokens.max()) < self.vocab:
            raise ValueError(f'{what} holds a token outside the vocabulary')
        return tokens.to(self.device, torch.long).contiguous()

    def add_request(self, request, *, prompt=None, output=None, repetition=1.0, frequency=0.0, presence=0.0,
                    bias=None):
        """Take a free slot for ``request``. ``prompt`` / ``output``: its prompt tokens and the
        tokens emitted so far (ids on the host, or integer tensors; on-device ids outside the
        vocabulary are skipped and flagged in the device status). ``bias``: {token: value},
        or (ids, values) whose duplicates add in order (on-device ids outside the vocabulary
        are skipped). Returns the slot."""
        if not isinstance(request, str) or not request or request in self._slots:
            raise ValueError('Require a fresh nonempty request name')
        if not self._free:
            raise ValueError('Control slots exhausted')
        repetition, frequency, presence = float(repetition), float(frequency), float(presence)
        if not (math.isfinite(repetition) and repetition > 0 and math.isfinite(frequency) and math.isfinite(presence)):
            raise ValueError('repetition must be finite and positive, frequency and presence finite')
        prompt, output = self._ids(prompt, 'prompt'), self._ids(output, 'output')
        ids = values = None
        if bias is not None:
            ids, values = (list(bias.keys()), list(bias.values())) if isinstance(bias, dict) else bias
            ids = self._ids(ids, 'bias')
            values = torch.as_tensor(values, dtype=torch.float32).to(self.device)
            if values.shape != ids.shape or ids.numel() > self.max_bias:
                raise ValueError(f'bias: one value per token and at most max_bias = {self.max_bias} entries required')
        slot = self._free[0]
        self.counts[slot].zero_()
        self.prompt_bits[slot].zero_()
        n_bias = 0 if ids is None else ids.numel()
        # one upload: the penalties' bits, the bias count, the slot and the two token ranges
        host = torch.tensor([repetition, frequency, presence], dtype=torch.float32).view(torch.int32).tolist()
        words = _upload(host + [n_bias, slot, 0, prompt.numel(), 0, output.numel()], self.device)
        self.penalties[slot].copy_(words[:3].view(torch.float32))
        self.bias_len[slot:slot + 1].copy_(words[3:4])
        if n_bias:
            self.bias_ids[slot, :n_bias].copy_(ids)
            self.bias_values[slot, :n_bias].copy_(values)
        for tokens, cu, to_counts in ((prompt, words[5:7], False), (output, words[7:9], True)):
            if tokens.numel():
                self._add(tokens, cu, None, words[4:5], to_counts)
        self._slots[request] = self._free.pop(0)       # taken once its tables are filled
        return slot

    def remove_request(self, request):
        if request not in self._slots:
            raise KeyError(request)
        self._free.append(self._slots.pop(request))
        self._free.sort()

    def slot_index(self, requests):
        """int32 device tensor of the requests' slots, for the kernels' ``slots`` argument."""
        for r in requests:
            if r not in self._slots:
                raise KeyError(r)
        return _upload([self._slots[r] for r in requests], self.device)

    def _add(self, tokens, cu, n, slots, to_counts):
        with _on_device(self.device):
            _lib.check(_lib.load_library().dspark_control_tokens(
                tokens.data_ptr(), tokens.numel(), cu.data_ptr(), None if n is None else n.data_ptr(),
                slots.data_ptr(), slots.numel(), self.vocab, self.slots,
                self.counts.data_ptr() if to_counts else None, self.counts.stride(0),
                None if to_counts else self.prompt_bits.data_ptr(), self.prompt_bits.stride(0),
                _stream(self.device)), 'dspark_control_tokens')

    def commit(self, slots, emitted, cu_query, n_commit=None):
        """Count a round's emitted tokens: request i's are ``emitted[cu_query[i] ..]``, the first
        ``n_commit[i]`` of them (all without ``n_commit``); ``greedy_accept``'s outputs as they
        are. Device tensors, no host read: capturable."""
        r = slots.numel()
        if (slots.dtype != torch.int32 or slots.shape != (r,) or emitted.dtype != torch.long or emitted.ndim != 1
                or not emitted.is_contiguous() or cu_query.dtype != torch.int32 or cu_query.shape != (r + 1,)
                or (n_commit is not None and (n_commit.dtype != torch.int32 or n_commit.shape != (r,)))
                or any(t.device != self.device or not t.is_contiguous()
                       for t in (slots, emitted, cu_query) + (() if n_commit is None else (n_commit,)))):
            raise ValueError('commit: contiguous int32 [R] slots, int64 [N] emitted, int32 [R + 1] cu_query and int32 '
                             '[R] n_commit on the tables\' device required')
        self._add(emitted, cu_query, n_commit, slots, True)


def _arguments(logits, controls, slots, cu_query, tokens, masks, mask_index):
    device, vocab = controls.device, controls.vocab
    if (not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.dtype not in _DTYPES
            or logits.device != device or logits.requires_grad):
        raise ValueError("logits must be no-autograd bf16/fp32 [N, vocab] rows on the tables' device")
    (n, columns), (ld, step) = logits.shape, logits.stride()
    if columns != vocab or step != 1 or (n > 1 and ld < vocab):
        raise ValueError('logits must have vocab columns with unit stride and rows that do not overlap')
    r = slots.numel()
    if slots.dtype != torch.int32 or slots.ndim != 1 or slots.device != device or not slots.is_contiguous() or r < 1:
        raise ValueError("slots must be contiguous int32 [R] on the tables' device")
    cu = token = mask = index = None
    ld_mask = num_masks = 0
    if cu_query is None:
        if n != r or tokens is not None:
            raise ValueError('Without cu_query there is one row per request, and no proposals')
    else:
        if (cu_query.dtype != torch.int32 or cu_query.ndim != 1 or len(cu_query) != r + 1
                or cu_query.device != device or not cu_query.is_contiguous()):
            raise ValueError("cu_query must be contiguous int32 [R + 1] on the tables' device")
        cu = cu_query.data_ptr()
    if tokens is not None:
        if (tokens.dtype != torch.long or tokens.ndim != 1 or len(tokens) != n or tokens.device != device
                or not tokens.is_contiguous()):
            raise ValueError("tokens must be contiguous int64 [N] on the tables' device")
        token = tokens.data_ptr()
    if (masks is None) != (mask_index is None):
        raise ValueError('masks and mask_index go together')
    if masks is not None:
        words = controls.words
        if (masks.dtype != torch.int32 or masks.ndim != 2 or masks.device != device
                or mask_index.dtype != torch.int32 or mask_index.ndim != 1 or len(mask_index) != n
                or mask_index.device != device or not mask_index.is_contiguous()):
            raise ValueError("masks must be int32 [M, ceil(vocab / 32)] and mask_index int32 [N] on the tables' device")
        (num_masks, wide), (ld_mask, step) = masks.shape, masks.stride()
        if num_masks < 1 or wide < words or step != 1 or (num_masks > 1 and ld_mask < words):
            raise ValueError('masks must have ceil(vocab / 32) words a row with unit stride')
        ld_mask = max(ld_mask, words)
        mask, index = masks.data_ptr(), mask_index.data_ptr()
    return (logits.data_ptr(), max(ld, vocab), _DTYPES[logits.dtype], n, vocab, cu, token, slots.data_ptr(), r,
            *controls._table_args, mask, ld_mask, num_masks, index)


def control_logits(logits, controls, slots, *, cu_query=None, tokens=None, masks=None, mask_index=None,
                   mask_value=float('-inf'), out=None, out_dtype=None, flag_empty=False):
    """Controlled logits of a verify round or decode step (``dspark_control_logits``).

    ``logits`` [N, vocab] bf16/fp32 (rows may be strided); ``slots`` int32 [R] from
    ``controls.slot_index``; ``cu_query`` int32 [R + 1] the requests' rows (without it: one row
    per request); ``tokens`` int64 [N] the verified chunks (anchor, then proposals), as in
    ``greedy_accept``. ``masks`` int32 [M, ceil(vocab / 32)] grammar masks (bit set: allowed)
    and ``mask_index`` int32 [N] the row of each logits row, -1 for none. Returns [N, vocab] in
    ``out_dtype`` (the logits' dtype or float32); ``out=logits`` changes them in place.
    ``mask_value`` replaces forbidden logits: a finite one (``torch.finfo(dtype).min``) keeps
    the rows acceptable to ``stochastic_accept``, which refuses infinities. A row whose mask
    allows nothing is ``mask_value`` throughout, and sampling from it gives any token: with
    ``flag_empty`` such a row sets the device status bit ``DEVICE_EMPTY_MASK`` (one more small
    launch). Rows outside every request are not written."""
    args = _arguments(logits, controls, slots, cu_query, tokens, masks, mask_index)
    device, ld_out = controls.device, controls.vocab
    if out is None:
        if out_dtype is not None and out_dtype != logits.dtype and out_dtype != torch.float32:
            raise ValueError("out_dtype must be the logits' dtype or float32")
        out = torch.empty_like(logits, dtype=out_dtype, memory_format=torch.contiguous_format)
    else:
        if (out.shape != logits.shape or out.device != device or out.stride(1) != 1
                or (len(out) > 1 and out.stride(0) < ld_out) or (out_dtype is not None and out.dtype != out_dtype)
                or (out.dtype != logits.dtype and out.dtype != torch.float32)):
            raise ValueError("out must be [N, vocab] rows of the logits' dtype or float32 on their device")
        ld_out = max(out.stride(0), ld_out)
    with _on_device(device):
        _lib.check(_lib.load_library().dspark_control_logits(
            *args, float(mask_value), out.data_ptr(), ld_out, _DTYPES[out.dtype], _stream(device)),
            'dspark_control_logits')
        if flag_empty and masks is not None:
            # masks, ld_mask, num_masks, mask_index; rows and vocab; cu_q; requests
            _lib.check(_lib.load_library().dspark_control_check_masks(*args[-4:], args[3], args[4], args[5], args[8],
                                                                      _stream(device)), 'dspark_control_check_masks')
    return out


def control_argmax(logits, controls, slots, *, cu_query=None, tokens=None, masks=None, mask_index=None):
    """Index of each row's largest controlled logit, int32 [N] (``dspark_control_argmax``): the
    arguments of ``control_logits``, nothing written but the indices. Ties give the lowest
    index, NaN is largest, and a row whose mask allows nothing gives -1 and sets the
    device status bit ``DEVICE_EMPTY_MASK``. Rows outside every request stay unset."""
    args = _arguments(logits, controls, slots, cu_query, tokens, masks, mask_index)
    lib, device = _lib.load_library(), controls.device
    with _on_device(device):
        n = len(logits)
        nbytes = lib.dspark_control_argmax_scratch_bytes(n, controls.vocab)
        # one allocation: 8-byte partial maxima, then the indices
        scratch = controls.bias_len.new_empty(nbytes // 4 + n)
        pred = scratch[nbytes // 4:]
        _lib.check(lib.dspark_control_argmax(*args, pred.data_ptr(), scratch.data_ptr(), nbytes, _stream(device)),
                   'dspark_control_argmax')
    return pred
