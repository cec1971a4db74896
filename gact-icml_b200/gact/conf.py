"""Global configuration and the optimisation-level presets (reference: gact/gact/conf.py:1-72).

The presets mutate the shared ``config`` object exactly as the reference does; fields a preset does not
name keep their previous value (so, as in the reference, ``L3`` followed by ``L1`` leaves ``swap`` on).
``reset()`` is an addition for callers who want a clean slate between runs.
"""


class QuantizationConfig:
    def __init__(self):
        self.reset()

    def reset(self):
        # compress activations; False at level L0
        self.compress_activation = True
        # ---- general quantization setting ----
        # average number of bits per activation element (with auto precision) or the fixed width
        self.bit = 4
        self.group_size = 256
        # store identical saved tensors once (keyed by sampled values); costs a host sync per tensor
        self.check_dup = False
        # ---- auto precision ----
        self.auto_prec = True
        self.max_bit = 32
        self.adapt_interval = 1000
        self.work_dir = "./log/"
        self.log_interval = -1
        self.debug = False
        # ---- memory management ----
        self.swap = False
        self.prefetch = False
        # ---- additions of this implementation (the reference has no equivalent) ----
        # Where the rounding noise comes from.  'fast' (default): Philox4x32-7, one call per 16 elements, 8 bits of
        # noise each - the arithmetic is the reference's, the stream is not.  'curand': the reference's exact
        # stream (one generator per packed byte), bit-identical codes for the same seed, about 1.6x slower.
        # 'rtn': round to nearest, no noise.
        self.rng_mode = "fast"
        # fp32 only: evaluate (x-min)*scale+noise as one fused multiply-add, as the reference binary does
        self.fma = True
        # compress bfloat16 saved tensors too (the reference skips them: gact/gact/quantizer.py:57-58)
        self.quantize_bf16 = True
        # pack torch.bool saved tensors (dropout masks of current PyTorch) to 1 bit without any check
        self.pack_bool_masks = True
        # compress dense permuted views (transposed attention tensors) in memory order instead of copying them to
        # logical order first; the reconstruction keeps the source's strides
        self.keep_layout = True
        # share one payload between saves of the same, unmodified tensor object (found by identity and version
        # counter, no device read-back; the reference's check_dup fingerprints values instead and is off by default)
        self.dedup_saved = True
        # data-parallel probes: 'allreduce' = sensitivities of the all-reduced gradient (what the reference
        # computes under DDP); 'local' = probe without gradient all-reduce and sum the statistics instead;
        # 'shard' = like 'local', but every rank probes only its 1/W share of the tensors (W times fewer passes)
        self.dp_probe = "allreduce"
        # run the per-tensor part of the hooks in the native module gact/_hooks.so when it was built (same
        # decisions, same dictionaries, about half the host time per saved tensor); False = the Python code
        self.native_hooks = True
        # the 8-bit checkpoints of gact.layers: False = round to nearest, True = stochastically (unbiased)
        self.stochastic_checkpoints = False


def set_optimization_level(level):
    if level == 'L0':          # no compression
        config.compress_activation = False
    elif level == 'L1':        # fixed 4 bit
        config.auto_prec = False
        config.bit = 4
    elif level == 'L1.1':      # fixed 8 bit
        config.auto_prec = False
        config.bit = 8
    elif level == 'L1.2':      # fixed 2 bit
        config.auto_prec = False
        config.bit = 2
    elif level == 'L2':        # auto precision, 4 bit on average
        config.auto_prec = True
        config.bit = 4
    elif level == 'L2.1':      # auto precision, 3 bit on average
        config.auto_prec = True
        config.bit = 3
    elif level == 'L2.2':      # auto precision, 2 bit on average
        config.auto_prec = True
        config.bit = 2
    elif level == 'L3':        # auto precision 4 bit + swap to host memory
        config.auto_prec = True
        config.bit = 4
        config.swap = True
        config.prefetch = True
    elif level == 'swap':      # swap uncompressed tensors
        config.swap = True
        config.compress_activation = False
    elif level == 'L4bit-swap':  # fixed 4 bit + swap
        config.bit = 4
        config.swap = True
        config.prefetch = True
        config.auto_prec = False
    else:
        raise ValueError("Invalid level: " + level)


def set_adapt_interval(i):
    config.adapt_interval = i


config = QuantizationConfig()
