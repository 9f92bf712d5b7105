"""AdamW over many tensors at once, with the moments in 32 or in 8 bits (``csrc/adamw.hip``).

``AdamW`` is the optimizer object (``keras.pipeline``'s ``'adamw'`` and ``'adamw_8bit'``), ``adamw_step`` the same update as
a plain call on lists of tensors.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from . import _ops
from ._ops import _ptr, _raw_stream, _stream, require_device

QBLOCK = 128                          # TFR_ADAMW_QBLOCK: elements that share a scale
_MAX_TENSORS, _MAX_TENSORS_8 = 88, 64  # TFR_ADAMW_MAX_TENSORS, TFR_ADAMW8_MAX_TENSORS: tensors of one launch
_MAX_LAUNCH = 1 << 35                 # elements of one launch
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # TFR_DTYPE_*


def quantized_size(numel: int) -> Tuple[int, int]:
    """(codes, scales) of an 8-bit moment of ``numel`` elements: whole blocks."""
    blocks = -(-int(numel) // QBLOCK)
    return blocks * QBLOCK, blocks


def _check_hyper(lr, betas, eps, weight_decay):
    if not torch.is_tensor(lr) and not lr >= 0.0:
        raise ValueError('Invalid learning rate: {}'.format(lr))
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError('Invalid betas: {}'.format(betas))
    if not eps >= 0.0:
        raise ValueError('Invalid epsilon value: {}'.format(eps))
    if not weight_decay >= 0.0:
        raise ValueError('Invalid weight_decay value: {}'.format(weight_decay))


def _check_dense(t, like, numel, dtype, name):
    if t.dtype is not dtype or t.numel() != numel or t.get_device() != like.get_device() or not t.is_contiguous():
        raise ValueError('%s must be a dense %s tensor of %d elements on %s, got %s of shape %s on %s'
                         % (name, dtype, numel, like.device, t.dtype, tuple(t.shape), t.device))


def _uniform(params, grads, exp_avgs, exp_avg_sqs, eight):
    """The addresses of tensors of one device and type, all of them as they have to be; None where a closer look is needed
    (``_grouped``: several devices or types, nothing in a tensor, or something to refuse).  Whole lists at a time: a tower's
    14 tensors go in 25 us with the launch, 31 one by one."""
    T = torch.Tensor
    lists = [params, grads]
    for moments in (exp_avgs, exp_avg_sqs):
        if not eight:
            lists.append(moments)
        elif all(isinstance(x, (tuple, list)) and len(x) == 2 for x in moments):
            lists += zip(*moments)
        else:
            return None
    try:
        device, dtype = params[0].get_device(), params[0].dtype
        wanted = [dtype, dtype] + ([torch.int8, torch.float32, torch.uint8, torch.float32] if eight else [torch.float32] * 2)
        sizes = list(map(T.numel, params))
        fit = [sizes] * 4
        if eight:
            scales = [-(-n // QBLOCK) for n in sizes]
            codes = [n * QBLOCK for n in scales]
            fit = [sizes, sizes, codes, scales, codes, scales]
        for ts, d, n in zip(lists, wanted, fit):
            if ({t.dtype for t in ts} != {d} or set(map(T.get_device, ts)) != {device} or not all(map(T.is_contiguous, ts))
                    or list(map(T.numel, ts)) != n):
                return None
        columns = [list(map(T.data_ptr, ts)) for ts in lists]
    except (TypeError, AttributeError):
        return None
    if (device < 0 or dtype not in _DTYPES or min(sizes) == 0 or max(sizes) >= _MAX_LAUNCH
            or len(set().union(columns[0], *columns[2:])) != len(sizes) * (len(columns) - 1)
            or (eight and any((a | b) & 7 for a, b in zip(columns[2], columns[4])))):
        return None
    return {(device, dtype): columns + [sizes]}


def _grouped(params, grads, exp_avgs, exp_avg_sqs, eight):
    """By (device, type), the addresses of every tensor that holds something: columns of params, grads, exp_avgs, exp_avg_sqs (8
    bits: codes and scales of both), and of their numbers of elements."""
    groups, seen = {}, set()
    for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
        device, dtype, numel = p.get_device(), p.dtype, p.numel()
        if device < 0:
            require_device(p, 'params')
        if dtype not in _DTYPES:
            raise ValueError('params must be float32, bfloat16 or float16, got %s' % dtype)
        if not p.is_contiguous():
            raise ValueError('params must be dense, got strides %s' % (p.stride(),))
        _check_dense(g, p, numel, dtype, 'grads')
        if isinstance(m, (tuple, list)) != eight or isinstance(v, (tuple, list)) != eight:
            raise ValueError('moments of 8 and of 32 bits in one call')
        if eight:
            codes, blocks = quantized_size(numel)
            _check_dense(m[0], p, codes, torch.int8, 'exp_avgs codes')
            _check_dense(m[1], p, blocks, torch.float32, 'exp_avgs scales')
            _check_dense(v[0], p, codes, torch.uint8, 'exp_avg_sqs codes')
            _check_dense(v[1], p, blocks, torch.float32, 'exp_avg_sqs scales')
            row = (p.data_ptr(), g.data_ptr(), m[0].data_ptr(), m[1].data_ptr(), v[0].data_ptr(), v[1].data_ptr(), numel)
            if (row[2] | row[4]) & 7:
                raise ValueError('codes must be 8-byte aligned')
        else:
            _check_dense(m, p, numel, torch.float32, 'exp_avgs')
            _check_dense(v, p, numel, torch.float32, 'exp_avg_sqs')
            row = (p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), numel)
        if numel >= _MAX_LAUNCH:
            raise ValueError('params of at most %d elements, got %d' % (_MAX_LAUNCH - 1, numel))
        if numel:
            if not seen.isdisjoint(row[2:-1] + row[:1]) or len(set(row[2:-1] + row[:1])) < len(row) - 2:
                raise ValueError('the same parameter or moment twice')
            seen.update(row[2:-1] + row[:1])
            groups.setdefault((device, dtype), []).append(row)
    return {key: list(zip(*rows)) for key, rows in groups.items()}


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence, exp_avg_sqs: Sequence, *, step: int,
               lr: float, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               now: Optional[torch.Tensor] = None) -> None:
    """One AdamW step, in place, on all tensors: ``TFR_ADAMW_MAX_TENSORS`` tensors a launch.

    ``params`` / ``grads``: dense tensors of one type (float32, bfloat16, float16) a pair.  ``exp_avgs`` / ``exp_avg_sqs``:
    float32 tensors of the parameter's size, or all of them pairs ``(codes, scales)``: int8 / uint8 codes and float32 scales
    of ``quantized_size(param.numel())`` elements.  Parameters and moments are written: no two may share memory (two that begin
    at one address are refused).  ``step`` counts from 1.  ``now``: float32 ``[3]`` on the device, the coefficients of a step
    that is counted there, as ``tfr_adamw_advance`` writes them (``step`` and ``lr`` are then not used)."""
    n = len(params)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n):
        raise ValueError('lists of %d params, %d grads, %d exp_avgs and %d exp_avg_sqs' % (n, len(grads), len(exp_avgs), len(exp_avg_sqs)))
    _check_hyper(lr, betas, eps, weight_decay)
    if torch.is_tensor(lr):
        if now is None:
            raise ValueError('lr must be a number: a learning rate on the device needs a step that is counted there')
        lr = 0.0
    if now is None and step < 1:
        raise ValueError('step counts from 1, got %r' % (step,))
    if n == 0:
        return
    if now is not None:
        _check_dense(now, params[0], 3, torch.float32, 'now')
        if any(p.get_device() != now.get_device() for p in params):
            raise ValueError('now is on %s: a step that is counted on a device takes the parameters of that device' % (now.device,))
    tail = (lr, betas[0], betas[1], eps, weight_decay, step, None if now is None else now.data_ptr())
    for launch, name, device, args, _ in _launches(params, grads, exp_avgs, exp_avg_sqs, False):
        with _ops.device_of(device):
            rc = launch(*args, *tail, _raw_stream(device))
        if rc:
            _lib.check(rc, name)
    _changed(params)


def _launches(params, grads, exp_avgs, exp_avg_sqs, counted):
    """(C entry point, its name, device, first arguments, addresses of the parameters) of every launch of a step."""
    eight = isinstance(exp_avgs[0], (tuple, list))
    groups = _uniform(params, grads, exp_avgs, exp_avg_sqs, eight) or _grouped(params, grads, exp_avgs, exp_avg_sqs, eight)
    cap = _MAX_TENSORS_8 if eight else _MAX_TENSORS
    name = ('tfr_adamw8' if eight else 'tfr_adamw') + ('_counted' if counted else '')
    launch = getattr(_lib.load(), name)
    for (device, dtype), columns in groups.items():
        sizes, at = columns[-1], 0
        while at < len(sizes):
            end = min(at + cap, len(sizes))
            while sum(sizes[at:end]) >= _MAX_LAUNCH:
                end -= 1
            addresses = ctypes.c_void_p * (end - at)
            yield (launch, name, device, (_DTYPES[dtype], end - at, *[addresses(*c[at:end]) for c in columns[:-1]],
                                          (ctypes.c_int64 * (end - at))(*sizes[at:end])), columns[0][at:end])
            at = end


def _changed(params):
    """A graph that saved a parameter must not go backward any more."""
    try:
        torch.autograd.graph.increment_version(params)
    except RuntimeError:                                       # inference tensors have no version
        for p in params:
            if not p.is_inference():
                torch.autograd.graph.increment_version(p)


def _counted_step(params, grads, exp_avgs, exp_avg_sqs, steps, all_steps, lr, betas, eps, weight_decay):
    """``adamw_step`` with the step counts on the device: ``steps`` one int64 tensor a parameter, ``all_steps`` one that counts
    the calls; ``lr`` a number or a float32 tensor of one element there."""
    lr_device = lr.data_ptr() if torch.is_tensor(lr) else None
    tail = (0.0 if lr_device else lr, betas[0], betas[1], eps, weight_decay)
    count_of = {p.data_ptr(): t.data_ptr() for p, t in zip(params, steps)}
    every = all_steps.data_ptr()
    for launch, name, device, args, addresses in _launches(params, grads, exp_avgs, exp_avg_sqs, True):
        with _ops.device_of(device):
            now = torch.empty(3 * len(addresses), dtype=torch.float32, device=all_steps.device)
            counts = (ctypes.c_void_p * len(addresses))(*[count_of[a] for a in addresses])
            rc = launch(*args, counts, every, lr_device, *tail, now.data_ptr(), _raw_stream(device))
        if rc:
            _lib.check(rc, name)
        every = None
    _changed(params)


def _dequantize(codes, scales, dtype, square):
    require_device(codes, 'codes')
    if codes.dtype != dtype or codes.numel() % QBLOCK or not codes.is_contiguous():
        raise ValueError('codes must be dense %s in whole blocks of %d, got %s of shape %s' % (dtype, QBLOCK, codes.dtype, tuple(codes.shape)))
    _check_dense(scales, codes, codes.numel() // QBLOCK, torch.float32, 'scales')
    if codes.data_ptr() & 7:
        raise ValueError('codes must be 8-byte aligned')
    out = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
    _lib.check(_lib.load().tfr_adamw_dequantize(_ptr(codes), _ptr(scales), codes.numel(), int(square), _ptr(out), _stream()),
               'tfr_adamw_dequantize')
    return out


@_ops.device_guarded
def dequantize_exp_avg(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 first moments that int8 codes stand for: code * scale (-128: NaN)."""
    return _dequantize(codes, scales, torch.int8, False)


@_ops.device_guarded
def dequantize_exp_avg_sq(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 second moments that uint8 codes stand for: (code * scale)^2."""
    return _dequantize(codes, scales, torch.uint8, True)


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over dense float32, bfloat16 or float16 parameters, one launch per
    ``TFR_ADAMW_MAX_TENSORS`` tensors.

    ``state_bits=8`` holds the moments in 8 bits (2.06 bytes an element for both instead of 8).  ``capturable=True`` counts the
    steps on the device (one small launch more), so that a step recorded in a hipGraph keeps counting when it is replayed;
    ``lr`` may then be a float32 device tensor of one element.  Either way every parameter has its own count
    (``state[p]['step']``): one that gets its first gradient late is corrected by the steps that it took itself.  The state is
    made by the first eager step (or by ``init_state()``); a capture needs it to be there."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, capturable=False):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      capturable=capturable))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            _check_hyper(g['lr'], g['betas'], g['eps'], g['weight_decay'])
            if g['state_bits'] not in (8, 32):
                raise ValueError('state_bits must be 8 or 32, got {}'.format(g['state_bits']))
            if torch.is_tensor(g['lr']) and not g['capturable']:
                raise ValueError('lr as a tensor needs capturable=True')
        except ValueError:
            self.param_groups.pop()
            raise

    def _state_of(self, p, group):
        s = self.state[p]
        there = torch.is_tensor(s.get('step'))                 # counted on the device
        if 'exp_avg' in s and there == group['capturable']:
            return s
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('AdamW: the state must be there before a stream capture (run a step or init_state() first)')
        require_device(p, 'params')
        if 'exp_avg' not in s:
            if group['state_bits'] == 32:
                s['exp_avg'] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                s['exp_avg_sq'] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            else:
                codes, blocks = quantized_size(p.numel())
                s['exp_avg'] = torch.zeros(codes, dtype=torch.int8, device=p.device)
                s['exp_avg_sq'] = torch.zeros(codes, dtype=torch.uint8, device=p.device)
                s['exp_avg_scale'] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
                s['exp_avg_sq_scale'] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        taken = int(s.get('step', 0))                          # `capturable` may have been switched
        s['step'] = torch.full((1,), taken, dtype=torch.int64, device=p.device) if group['capturable'] else taken
        return s

    def _counter(self, group, device):
        """The steps of a capturable group, on the device (its parameters count their own)."""
        if group.get('step_count') is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError('AdamW: the state must be there before a stream capture (run a step or init_state() first)')
            group['step_count'] = torch.zeros(1, dtype=torch.int64, device=device)
        return group['step_count']

    def init_state(self) -> None:
        """Makes the state of every parameter (before a stream capture without an eager step)."""
        for group in self.param_groups:
            for p in group['params']:
                self._state_of(p, group)
            if group['capturable'] and group['params']:
                self._counter(group, group['params'][0].device)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            eight, there = group['state_bits'] == 8, group['capturable']
            counted_by = torch.Tensor if there else int
            runs = {}                                          # by step count: parameters that were frozen for a while have their own
            for p in group['params']:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError('AdamW does not take sparse gradients')
                s = self.state[p]
                if type(s.get('step')) is not counted_by:
                    s = self._state_of(p, group)
                t = 0 if there else s['step'] + 1
                m, v = s['exp_avg'], s['exp_avg_sq']
                runs.setdefault(t, []).append((s, p, p.grad.contiguous(), (m, s['exp_avg_scale']) if eight else m,
                                               (v, s['exp_avg_sq_scale']) if eight else v))
            if not runs:
                continue
            how = dict(lr=group['lr'], betas=group['betas'], eps=group['eps'], weight_decay=group['weight_decay'])
            if there:                                          # all in one list: the launches read the counts on the device
                states, p, g, m, v = zip(*runs[0])
                count = self._counter(group, p[0].device)
                if any(q.device != count.device for q in group['params']):
                    raise ValueError('AdamW: a capturable group lives on one device')
                lr = group['lr']
                if torch.is_tensor(lr) and not (lr.is_cuda and lr.dtype == torch.float32 and lr.numel() == 1 and lr.device == count.device):
                    raise ValueError('lr must be a float32 tensor of one element on %s' % (count.device,))
                _check_hyper(**how)
                _counted_step(p, g, m, v, [s['step'] for s in states], count, **how)
                continue
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError('AdamW: a step inside a stream capture needs capturable=True (the step count would be frozen)')
            for t, items in runs.items():
                states, p, g, m, v = zip(*items)
                adamw_step(p, g, m, v, step=t, **how)
                for s in states:                               # counted once it is launched: a step that is refused is none
                    s['step'] = t
        return loss

    def _moments(self, p, group):
        """(type, elements) of what the state of a parameter holds beside its count."""
        if group['state_bits'] == 32:
            return {'exp_avg': (torch.float32, p.numel()), 'exp_avg_sq': (torch.float32, p.numel())}
        codes, blocks = quantized_size(p.numel())
        return {'exp_avg': (torch.int8, codes), 'exp_avg_sq': (torch.uint8, codes), 'exp_avg_scale': (torch.float32, blocks),
                'exp_avg_sq_scale': (torch.float32, blocks)}

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Loads what ``state_dict`` gave; a state that does not fit raises and changes nothing.  Moments keep their own types
        (the base class would cast them to the parameter's).  Tensors that are there already -- moments, counts, a learning
        rate on the device -- stay and are filled, with zeros where the loaded state holds none: a captured step goes on with
        them, and a group that is capturable stays so."""
        saved, mine = state_dict['param_groups'], [dict(g) for g in self.param_groups]
        held = {p: dict(s) for p, s in self.state.items()}
        for group, given in zip(mine, saved):
            if group['capturable'] and given['state_bits'] != group['state_bits'] and any(held.get(p) for p in group['params']):
                raise ValueError('a state of %d bits does not fit one of %d that a captured step may hold' % (given['state_bits'], group['state_bits']))
            for p, i in zip(group['params'], given['params']):
                for key, (dtype, numel) in self._moments(p, given).items() if state_dict['state'].get(i) else ():
                    value = state_dict['state'][i].get(key)
                    if not torch.is_tensor(value) or value.numel() != numel or (value.dtype != dtype if given['state_bits'] == 8 else not value.is_floating_point()):
                        raise ValueError('state %s does not fit a parameter of %d elements: %d of %s are wanted' % (key, p.numel(), numel, dtype))
        super().load_state_dict(state_dict)
        for group, old, given in zip(self.param_groups, mine, saved):
            group['capturable'] = there = bool(group['capturable'] or old['capturable'])
            count = given.get('step_count')
            for p, i in zip(group['params'], given['params']):
                self._fill_state(p, group, held.get(p, {}), state_dict['state'].get(i) or None, count)
            if not group['params']:
                continue
            device = group['params'][0].device
            group.pop('coefficients', None)                    # of a state that counted by group alone
            group.pop('step_count', None)
            have = old.get('step_count')
            if there and (count is not None or have is not None):
                group['step_count'] = _filled(have if have is not None and have.device == device else None, 0 if count is None else count, torch.int64, device)
            if torch.is_tensor(old['lr']):
                group['lr'] = _filled(old['lr'], group['lr'], old['lr'].dtype, device)
            elif torch.is_tensor(group['lr']):
                group['lr'] = group['lr'].to(device)

    def _fill_state(self, p, group, have, given, count):
        """The state of one parameter from the saved one (None: as before any step), in the tensors of ``have`` that fit."""
        moments = self._moments(p, group)
        have = {k: t for k, t in have.items() if torch.is_tensor(t) and t.device == p.device}
        fits = {k: t for k, t in have.items() if k in moments and (t.dtype, t.numel()) == moments[k]}
        if given is None:
            self.state.pop(p, None)
            if len(fits) < len(moments):
                return
        s = self.state[p] = {}
        for key, (dtype, _) in moments.items():
            s[key] = _filled(fits.get(key), 0 if given is None else given[key], dtype, p.device)
        # counted by group alone, each of its parameters took all of the group's steps
        taken = 0 if given is None else given.get('step', 0 if count is None else count)
        s['step'] = _filled(have.get('step'), taken, torch.int64, p.device) if group['capturable'] else int(taken)
        for key, value in (given or {}).items():
            if key not in s:
                s[key] = value


def _filled(have, value, dtype, device):
    """``value`` (a tensor or a number) in the tensor ``have``, or in a new one where there is none."""
    if not torch.is_tensor(value):
        return torch.full((1,), value, dtype=dtype, device=device) if have is None else have.fill_(value)
    if have is None:
        return value.to(device=device, dtype=dtype, copy=True)
    return have.copy_(value.reshape(have.shape))
