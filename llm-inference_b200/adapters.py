"""The low-rank adapters that a server's requests choose from, on the device.

:class:`AdapterSet` holds up to `n_adapters` adapters for one model shape, stacked per layer and projection as
``lora_add`` and ``lora_gate_up`` take them. An adapter comes from tensors (:meth:`AdapterSet.set`) or from a directory with
``adapter_config.json`` and ``adapter_model.safetensors`` (:meth:`AdapterSet.load`); projections that it does not have
are left alone.

    adapters = AdapterSet(weights.shape, n_adapters=8, rank=16)
    adapters.load(0, adapter_dir)
    server = PagedServer(weights, n_pages=4096, adapters=adapters)
    server.add(prompt, adapter=0)
"""
from __future__ import annotations

import json
import math
import struct
from pathlib import Path

import numpy as np

from .checkpoint import CheckpointError, Qwen3Shape
from .lora import LoraStack

# the calls of a layer: projections of one input
GROUPS = {"qkv": ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), "o": ("self_attn.o_proj",),
          "gate_up": ("mlp.gate_proj", "mlp.up_proj"), "down": ("mlp.down_proj",)}
PROJECTIONS = tuple(p for group in GROUPS.values() for p in group)


def projection_sizes(s: Qwen3Shape) -> dict[str, tuple[int, int]]:
    """(inputs, outputs) of each projection that can be adapted."""
    return {"self_attn.q_proj": (s.hidden_size, s.q_dim), "self_attn.k_proj": (s.hidden_size, s.kv_dim),
            "self_attn.v_proj": (s.hidden_size, s.kv_dim), "self_attn.o_proj": (s.q_dim, s.hidden_size),
            "mlp.gate_proj": (s.hidden_size, s.intermediate_size), "mlp.up_proj": (s.hidden_size, s.intermediate_size),
            "mlp.down_proj": (s.intermediate_size, s.hidden_size)}


def read_adapter(path, s: Qwen3Shape):
    """({(layer, projection): (A [r, inputs], B [outputs, r])} as torch tensors, scale) of an adapter's directory. Checks names,
    shapes, types and the options that change what an adapter computes."""
    import torch
    d = Path(path)
    cfg = json.loads((d / "adapter_config.json").read_text())
    if cfg.get("peft_type", "LORA") != "LORA":
        raise CheckpointError(f"adapter type {cfg.get('peft_type')!r}, expected 'LORA'")
    for key in ("use_dora", "use_qalora", "rank_pattern", "alpha_pattern", "modules_to_save", "layer_replication", "lora_bias",
                "alora_invocation_tokens", "arrow_config"):
        if cfg.get(key):
            raise CheckpointError(f"adapter_config.json: {key} is not supported")
    # of these A and B start beside the base's weights as they are; others take a part out of the base first
    if cfg.get("init_lora_weights") not in (None, True, False, "gaussian", "eva", "orthogonal"):
        raise CheckpointError(f"adapter_config.json: init_lora_weights {cfg['init_lora_weights']!r} belongs to a changed base; save it converted")
    if cfg.get("bias", "none") != "none":
        raise CheckpointError("adapter_config.json: biases are not supported")
    r, alpha = cfg.get("r"), cfg.get("lora_alpha")
    if not isinstance(r, int) or r < 1 or not isinstance(alpha, (int, float)) or not math.isfinite(alpha):
        raise CheckpointError("adapter_config.json needs an integer r and a number lora_alpha")
    scale = alpha / (math.sqrt(r) if cfg.get("use_rslora") else r)
    file = d / "adapter_model.safetensors"
    size = file.stat().st_size
    with open(file, "rb") as f:
        head = f.read(8)
        if len(head) < 8 or struct.unpack("<Q", head)[0] > size - 8:
            raise CheckpointError(f"{file}: bad header")
        (n,) = struct.unpack("<Q", head)
        header = json.loads(f.read(n))
    data = np.memmap(file, dtype=np.uint8, mode="r")[8 + n:]
    types = {"BF16": torch.bfloat16, "F16": torch.float16, "F32": torch.float32}
    found: dict[tuple[int, str], dict[str, object]] = {}
    sizes = projection_sizes(s)
    for name, meta in header.items():
        if name == "__metadata__":
            continue
        parts = name.split(".")
        try:
            at = parts.index("layers")
            layer, proj, which = int(parts[at + 1]), ".".join(parts[at + 2:at + 4]), parts[at + 4]
            if parts[at + 5:] != ["weight"] or which not in ("lora_A", "lora_B") or proj not in sizes or not 0 <= layer < s.num_hidden_layers:
                raise ValueError
        except (ValueError, IndexError):
            raise CheckpointError(f"tensor {name} has no place in this model") from None
        k, rows = sizes[proj]
        want = [r, k] if which == "lora_A" else [rows, r]
        if meta["shape"] != want or meta["dtype"] not in types:
            raise CheckpointError(f"{name}: {meta['dtype']} {meta['shape']}, expected {want}")
        b, e = meta["data_offsets"]
        dtype = types[meta["dtype"]]
        if b < 0 or e > len(data) or e - b != want[0] * want[1] * dtype.itemsize:
            raise CheckpointError(f"{name}: data_offsets do not match its shape")
        found.setdefault((layer, proj), {})[which] = torch.frombuffer(bytearray(data[b:e]), dtype=dtype).view(want)
    for (layer, proj), ab in found.items():
        if len(ab) != 2:
            raise CheckpointError(f"layer {layer} {proj} has only one of lora_A and lora_B")
    return {key: (ab["lora_A"], ab["lora_B"]) for key, ab in found.items()}, scale


class AdapterSet:
    """Device memory for `n_adapters` adapters of rank up to `rank` (a multiple of 8 up to 128). Setting an adapter is ordered
    with torch's current stream: requests that use the old one must have run on that stream or be done."""

    def __init__(self, shape: Qwen3Shape, n_adapters: int, rank: int = 16):
        import torch
        self.shape, self.n_adapters, self.rank = shape, n_adapters, rank
        sizes = projection_sizes(shape)
        self.scale = torch.zeros(n_adapters, dtype=torch.float32, device="cuda")
        self.loaded: set[int] = set()
        self._a, self._b, self._ranks = {}, {}, {}
        # per layer, the adapters that have one of gate and up
        self.with_gate_up: list[set[int]] = [set() for _ in range(shape.num_hidden_layers)]
        self.stacks: dict[str, list[LoraStack]] = {g: [] for g in GROUPS}
        for layer in range(shape.num_hidden_layers):
            for g, projs in GROUPS.items():
                ranks = self._ranks[layer, g] = torch.zeros(n_adapters, dtype=torch.int32, device="cuda")
                for p in projs:
                    k, n = sizes[p]
                    self._a[layer, p] = torch.zeros(n_adapters, rank, k, dtype=torch.bfloat16, device="cuda")
                    self._b[layer, p] = torch.zeros(n_adapters, n, rank, dtype=torch.bfloat16, device="cuda")
                self.stacks[g].append(LoraStack([self._a[layer, p] for p in projs], [self._b[layer, p] for p in projs], self.scale,
                                                ranks))

    def set(self, i: int, tensors, scale: float) -> None:
        """Adapter i from {(layer, projection): (A [r, inputs], B [outputs, r])}, replacing what it was. Ranks may differ between
        projections."""
        if not 0 <= i < self.n_adapters:
            raise ValueError(f"adapter {i} of {self.n_adapters}")
        sizes = projection_sizes(self.shape)
        for (layer, proj), (a, b) in tensors.items():  # before anything is written
            if proj not in sizes or not 0 <= layer < self.shape.num_hidden_layers:
                raise ValueError(f"no projection {proj!r} in layer {layer}")
            k, n = sizes[proj]
            if a.dim() != 2 or a.shape[0] < 1 or tuple(a.shape) != (b.shape[-1], k) or tuple(b.shape) != (n, a.shape[0]):
                raise ValueError(f"layer {layer} {proj}: A {tuple(a.shape)} and B {tuple(b.shape)}, expected [r, {k}] and [{n}, r]")
            if a.shape[0] > self.rank:
                raise ValueError(f"layer {layer} {proj}: rank {a.shape[0]}, the set holds {self.rank}")
        for layer in range(self.shape.num_hidden_layers):
            for g, projs in GROUPS.items():
                most = 0
                for p in projs:
                    a, b = self._a[layer, p][i], self._b[layer, p][i]
                    a.zero_()
                    b.zero_()
                    if (layer, p) in tensors:
                        ta, tb = tensors[layer, p]
                        most = max(most, ta.shape[0])
                        a[:ta.shape[0]].copy_(ta)
                        b[:, :ta.shape[0]].copy_(tb)
                self._ranks[layer, g][i] = most
            self.with_gate_up[layer].discard(i)
            if any((layer, p) in tensors for p in GROUPS["gate_up"]):
                self.with_gate_up[layer].add(i)
        self.scale[i] = scale
        self.loaded.add(i)

    def load(self, i: int, path) -> None:
        """Adapter i from a directory (:func:`read_adapter`)."""
        self.set(i, *read_adapter(path, self.shape))
