"""Benchmarks of the secondary configurations (the headline one is ``bench.py`` at the repository root):
``config3_gather`` (compressed-gradient gather), ``config4_tp`` (18B-class tensor-parallel window),
``config5_validator`` (validator scoring) and ``activation_modes`` (a micro-step in each mode of activation
checkpointing, scoring with 8-bit projections).  Each prints one JSON line per case."""
