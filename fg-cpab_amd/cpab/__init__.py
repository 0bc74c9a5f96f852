"""MI355X-native CPAB transformations (drop-in for FG-CPAB's ``cpab`` package), and the
operators of a network that reads signals and gives theta, with its optimiser's step."""
from .cpab import Cpab
from .pytorch.optim import AdamW, adamw_step
from .pytorch.sequence import gated_recurrence, rms_norm

__all__ = ['Cpab', 'gated_recurrence', 'rms_norm', 'adamw_step', 'AdamW']
