"""`komp.kv` is `comp_amd.kv`: this module replaces itself with it on import."""

import sys

from comp_amd import kv as _module

sys.modules[__name__] = _module
