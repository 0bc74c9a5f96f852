"""MI355X-native CPAB transformations (drop-in for FG-CPAB's ``cpab`` package), and the
operators of a network that reads signals and gives theta, with its optimiser's step."""
from .cpab import Cpab
from .pytorch.heads import gated_delta_rule, qk_norm
from .pytorch.optim import AdamW, Muon, adamw_step, muon_step
from .pytorch.sequence import gated_recurrence, rms_norm

__all__ = ['Cpab', 'gated_recurrence', 'gated_delta_rule', 'rms_norm', 'qk_norm', 'adamw_step', 'AdamW',
           'muon_step', 'Muon']
