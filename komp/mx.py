"""`komp.mx` is `comp_amd.mx`: this module replaces itself with it on import."""

import sys

from comp_amd import mx as _module

sys.modules[__name__] = _module
