"""AdamW over all parameters at once, with moments in 32 or 8 bits.  No counterpart in the reference;
the work is done by the HIP kernels behind `_C.adamw_step` and `_C.grad_norm`."""
import torch

from .. import _C


class AdamW(torch.optim.Optimizer):
    """Decoupled weight decay and bias-corrected moments, as the formula of _C.adamw_step says, in one
    launch for several dozen parameters (float32 or bfloat16, on one GPU).

    bits: of the moments, 32 or 8 (a quarter of the memory and a little over).
    max_norm: gradients are clipped by the norm of all of them, which the step reads while it
    updates: they are not changed themselves.  `grad_norm` holds the last step's norm.
    capturable: steps are counted on the GPU, so that a captured step can be replayed; a learning
    rate that changes between replays is a float32 value on the GPU then (a group's 'lr').  The first
    step, which makes the moments, is not captured.
    seed: of the rounding in 8 bits."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32,
                 max_norm=None, capturable=False, seed=0):
        self.max_norm, self.capturable, self.seed, self.grad_norm = max_norm, capturable, seed, None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      bits=bits))

    def add_param_group(self, param_group):
        if isinstance(param_group, dict) and param_group.get('bits', self.defaults['bits']) not in (32, 8):
            raise ValueError('Moments are held in 32 or 8 bits')
        super().add_param_group(param_group)

    def __getstate__(self):
        own = ('max_norm', 'capturable', 'seed', 'grad_norm')
        return dict(super().__getstate__(), **{name: getattr(self, name) for name in own})

    def _make(self, state, p, bits, counter):
        """The moments of a parameter, zeros when it first has a gradient."""
        zeros = {32: torch.float32, 8: torch.uint8}[bits]
        state['step'] = counter() if self.capturable else 0
        for name in ('first', 'second'):
            state[name] = torch.zeros(p.shape, dtype=zeros, device=p.device)
            if bits == 8:
                state[name + '_scale'] = torch.zeros(-(-p.numel() // _C.ADAMW_BLOCK), dtype=torch.float32,
                                                     device=p.device)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # (hundreds of parameters: each is looked at as rarely as can be.  The same gradient of several
        # parameters is read, and counts in the norm, once)
        dense, given = {}, []
        for group in self.param_groups:
            gradients = [p.grad for p in group['params']]
            given.append(gradients)
            for g in gradients:
                if g is not None and id(g) not in dense:
                    if g.is_sparse:
                        raise RuntimeError('AdamW does not support sparse gradients')
                    dense[id(g)] = g.contiguous()
        if not dense:
            return loss
        capturing = torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()
        if capturing:
            if not self.capturable:
                raise RuntimeError('Only a capturable AdamW counts the steps of a captured one')
            if any(g is not None and not self.state.get(p) for group, gradients in zip(self.param_groups, given)
                   for p, g in zip(group['params'], gradients)):
                raise RuntimeError('The first step of a parameter makes its moments and is not captured')
        norm = None
        if self.max_norm is not None:
            norm = self.grad_norm = _C.grad_norm(list(dense.values()))
        # (all are checked before the first changes anything: a step that is refused leaves all as it was)
        updates = []
        for group, gradients in zip(self.param_groups, given):
            made = []

            def counter():
                # parameters that first have gradients in the same call share a counter
                if not made:
                    made.append(torch.zeros((), dtype=torch.int64, device=group['params'][0].device))
                return made[0]

            alike, absent = {}, {}
            for p, g in zip(group['params'], gradients):
                if g is None:
                    if self.capturable and self.state.get(p):
                        absent.setdefault(id(self.state[p]['step']), []).append(self.state[p])
                    continue
                state = self.state[p]
                if not state:
                    self._make(state, p, group['bits'], counter)
                step = state['step']
                key = id(step) if self.capturable else step
                if key not in alike:
                    alike[key] = (step, [], [], [])
                _, params, grads, states = alike[key]
                params.append(p)
                grads.append(dense[id(g)])
                states.append(state)
            for key, (step, params, grads, states) in alike.items():
                if key in absent:  # whose counter stays behind
                    if capturing:
                        raise RuntimeError('Parameters without gradients share a counter with others: take '
                                           'a step without them before the captured one')
                    behind = step.clone()
                    for state in absent[key]:
                        state['step'] = behind
                updates.append(self._update(group, step, params, grads, states, norm, len(updates)))
        for update in updates:
            update()
        return loss

    def _update(self, group, step, params, grads, states, norm, call):
        """-> what changes parameters that share a count."""
        counted = isinstance(step, torch.Tensor)
        dense = list(map(torch.Tensor.contiguous, params))
        scales = {}
        if group['bits'] == 8:
            scales = dict(first_scales=[s['first_scale'] for s in states],
                          second_scales=[s['second_scale'] for s in states],
                          seed=self.seed + 0x9E3779B1 * call)
        number = step if counted else step + 1
        launch = _C._adamw_call(dense, grads, [s['first'] for s in states], [s['second'] for s in states], number,
                                group['lr'], group['betas'], group['eps'], group['weight_decay'], grad_norm=norm,
                                max_norm=None if norm is None else self.max_norm, **scales)

        def update():
            if counted:
                step.add_(1)
            try:
                launch()
            except RuntimeError:  # a step that is not launched is none
                if counted:
                    step.sub_(1)
                raise
            if not counted:
                for state in states:
                    state['step'] = number
            for changed, p in zip(dense, params):
                if changed is not p:
                    p.copy_(changed)
        return update

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # moments keep their own types (the base class casts them to the parameters')
        ids = [i for group in state_dict['param_groups'] for i in group['params']]
        for group in self.param_groups:
            if isinstance(group['lr'], torch.Tensor) and group['params']:
                group['lr'] = group['lr'].to(group['params'][0].device)
            counters = {}
            for p in group['params']:
                saved = state_dict['state'].get(ids.pop(0))
                if not saved:
                    continue
                state = {name: value.to(p.device, copy=True) for name, value in saved.items()
                         if name != 'step'}
                state['step'] = int(saved['step'])
                if self.capturable:  # as many counters in a group as there are numbers
                    if state['step'] not in counters:
                        counters[state['step']] = torch.tensor(state['step'], device=p.device)
                    state['step'] = counters[state['step']]
                self.state[p] = state
