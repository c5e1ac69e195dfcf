"""dhellam.operators.mx -> dhellam_amd.operators.mx."""
from dhellam_amd.operators.mx import *  # noqa: F401,F403
