"""Operator wrappers; same sub-packages as mamtorch/kernel/__init__.py:1-4 (v1 exact, v4 default), and ``encoder``: what an encoder
layer has beside its MAM layers."""
from . import v1
from . import v4
from . import encoder
