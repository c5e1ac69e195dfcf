"""dhellam.operators.grads -> dhellam_amd.operators.grads."""
from dhellam_amd.operators.grads import *  # noqa: F401,F403
