"""Sequential container (drop-in for triton_tagi/network.py).

``step(x, y, σ_v)`` runs forward → innovation → backward → capped update and
returns the pre-update predictions, exactly as the reference
(network.py:119-152). Two differences in *how*, not *what*:

* With ``fuse_update=True`` (default) each learnable layer applies its capped
  update inside its backward, right after propagating the deltas with the
  pre-update weights; the weight-gradient kernel then writes the parameters
  directly and no delta tensors are allocated. Every layer's update only
  touches its own parameters, so the result is the reference's
  backward-then-update. ``fuse_update=False`` keeps the reference's call
  structure (``delta_*`` tensors stored, ``update`` applied afterwards).
* Under data parallelism (``triton_tagi.distributed``) the batch sums of every
  layer are all-reduced before the update and the cap factor uses the global
  batch, so every replica applies the single-batch closed form.

``cuda_graph=True`` replays each step from a CUDA graph: the first step with a
new input shape (or σ_v) runs eagerly, the next one is captured on static input
buffers and replayed, and later steps copy their inputs in and replay. A step
of small layers is a few dozen short kernels, so launch overhead otherwise
dominates it. The replayed kernels are the eager step's; returned predictions
are copies. Under data parallelism the step is captured only if the reducer
says its collectives can be (``DataParallel(capturable=True)``, NCCL): the
graph then holds the SyncBN and gradient all-reduces too, every rank replays
the same graph, and the capture is thread-local so that the communicator's
watchdog thread may keep polling; otherwise the step runs eagerly. The
captured graph is keyed on the input shapes, σ_v, ``fuse_update`` and every
layer's training flag, so ``train()`` / ``eval()`` lead to a new capture.

``check_device=True`` (or the environment variable ``TAGI_B200_CHECK=1``) reads
the tensor-core kernels' error word after every step, or on a served network after
every forward pass that is not being captured (this synchronises), and raises
``RuntimeError`` if a bounded wait inside a kernel ran out, in which case that kernel's
outputs are incomplete.

``quantize()`` gives a network for serving: the same layers with every ``Linear`` (and
the projections of attention layers) in 8 bits, for ``forward`` only.
"""

from __future__ import annotations

import copy
import os

import torch
from torch import Tensor

from ._chain import backward_chain, forward_chain
from ._lib import check_device_status
from .base import LearnableLayer
from .layers.int8_linear import Int8Linear
from .layers.linear import Linear
from .layers.multihead_attention import MultiheadAttentionV2
from .layers.resblock import ResBlock
from .update.observation import compute_innovation
from .update.parameters import get_cap_factor


class Sequential:
    def __init__(self, layers: list, device="cuda", fuse_update: bool = True,
                 cuda_graph: bool = False, check_device: bool | None = None) -> None:
        self.device = torch.device(device)
        self.layers = layers
        self.fuse_update = fuse_update
        self.cuda_graph = cuda_graph
        if check_device is None:
            check_device = os.environ.get("TAGI_B200_CHECK", "0") == "1"
        self.check_device = check_device
        self._graph = None  # (key, CUDAGraph or None, static x, static y, outputs)
        self.reducer = None  # set by triton_tagi.distributed.DataParallel
        self.serving = False  # a network from quantize(): forward only
        for layer in self.layers:
            if isinstance(layer, ResBlock):
                layer.device = self.device
                for sub in layer._learnable:
                    self._move_layer_to_device(sub)
            elif isinstance(layer, LearnableLayer):
                self._move_layer_to_device(layer)
            if hasattr(layer, "running_mean"):
                layer.running_mean = layer.running_mean.to(self.device)
                layer.running_var = layer.running_var.to(self.device)

    def _move_layer_to_device(self, layer) -> None:
        if isinstance(layer, MultiheadAttentionV2):
            layer.device = self.device
            for sub in (layer.q_proj, layer.k_proj, layer.v_proj):
                self._move_layer_to_device(sub)
            return
        if getattr(layer, "mw", None) is None:
            return
        layer.device = self.device
        for name in ("mw", "Sw", "mb", "Sb", "running_mean", "running_var"):
            t = getattr(layer, name, None)
            if t is not None:
                setattr(layer, name, t.to(self.device))

    def learnable_layers(self) -> list[LearnableLayer]:
        return [layer for layer in self.layers if isinstance(layer, LearnableLayer)]

    def leaves(self) -> list[LearnableLayer]:
        """Learnable layers that own parameters, in network order."""
        out = []
        for layer in self.learnable_layers():
            out += layer._leaves()
        return out

    def forward(self, x: Tensor) -> tuple[Tensor, Tensor]:
        out = forward_chain(self.layers, x, torch.zeros_like(x))
        if (self.serving and self.check_device
                and not (x.is_cuda and torch.cuda.is_current_stream_capturing())):
            check_device_status()
        return out

    def quantize(self) -> "Sequential":
        """A network that serves this one's predictions from 8-bit weights: its ``Linear``
        layers and attention projections as they are now, laid out once (``Int8Linear``;
        those of more inputs than that takes stay in 32 bits).
        The other layers are copies that share their parameters with this network, and
        nothing else: passes of the two do not disturb one another. They are in eval mode:
        a BatchNorm2D serves with a copy of its running statistics as they are now.
        Quantize again after training on. Only ``forward`` works on it."""
        net = copy.copy(self)
        net.layers = [layer._serving() if isinstance(layer, Linear)
                      else layer.quantize() if isinstance(layer, MultiheadAttentionV2)
                      else layer._serving_copy() for layer in self.layers]
        net.serving, net.reducer, net._graph = True, None, None
        net.eval()
        return net

    def _refuse_serving(self) -> None:
        if self.serving:
            raise RuntimeError("a quantized network serves forward passes only; train the "
                               "network that it was made from")

    def step(self, x_batch: Tensor, y_batch: Tensor, sigma_v: float) -> tuple[Tensor, Tensor]:
        self._refuse_serving()
        red = self.reducer
        if self.cuda_graph and x_batch.is_cuda and (
                red is None or getattr(red, "capturable", False)):
            out = self._graph_step(x_batch, y_batch, sigma_v)
        else:
            out = self._step(x_batch, y_batch, sigma_v)
        if self.check_device:
            check_device_status()
        return out

    def _modes(self) -> tuple:
        """Training flags of every layer (and sub-layer), in network order."""
        flags = []

        def walk(layer):
            flags.append(getattr(layer, "training", None))
            for sub in getattr(layer, "_learnable", ()):
                if sub is not layer:
                    walk(sub)

        for layer in self.layers:
            walk(layer)
        return tuple(flags)

    def _graph_step(self, x_batch: Tensor, y_batch: Tensor, sigma_v: float) -> tuple[Tensor, Tensor]:
        key = (tuple(x_batch.shape), x_batch.dtype, tuple(y_batch.shape), y_batch.dtype,
               float(sigma_v), x_batch.device, self.fuse_update, self._modes())
        if self._graph is None or self._graph[0] != key:
            # first step of this shape: eager (it also leaves every layer in its
            # steady state, e.g. BatchNorm's running statistics initialised)
            self._graph = (key, None, None, None, None)
            return self._step(x_batch, y_batch, sigma_v)
        _, graph, sx, sy, out = self._graph
        if graph is None:
            sx, sy = x_batch.clone(), y_batch.clone()
            graph = torch.cuda.CUDAGraph()
            mode = "thread_local" if self.reducer is not None else "global"
            with torch.cuda.graph(graph, capture_error_mode=mode):
                out = self._step(sx, sy, sigma_v)
            self._graph = (key, graph, sx, sy, out)
        else:
            sx.copy_(x_batch)
            sy.copy_(y_batch)
        graph.replay()
        return out[0].clone(), out[1].clone()

    def _step(self, x_batch: Tensor, y_batch: Tensor, sigma_v: float) -> tuple[Tensor, Tensor]:
        red = self.reducer
        global_batch = x_batch.shape[0] * (red.world_size if red is not None else 1)
        y_pred_mu, y_pred_var = self.forward(x_batch)
        delta_mu, delta_var = compute_innovation(y_batch, y_pred_mu, y_pred_var, sigma_v)
        cap = get_cap_factor(global_batch)
        mode = "sums" if red is not None else ("update" if self.fuse_update else "deltas")
        learn = self.learnable_layers()
        for layer in learn:
            layer._set_param_mode(mode, cap, red)
        first = self.layers[0] if self.layers else None
        try:
            if red is not None:
                red.begin_step()
            if isinstance(first, LearnableLayer):
                first._skip_input_delta = True  # the input's deltas are not used
            delta_mu, delta_var = backward_chain(self.layers, delta_mu, delta_var)
            if red is not None:
                red.finish_step(cap)
            for layer in learn:
                layer.update(cap)
        finally:
            if isinstance(first, LearnableLayer):
                first._skip_input_delta = False
            for layer in learn:
                layer._set_param_mode("deltas")
        return y_pred_mu, y_pred_var

    def release_graph(self) -> None:
        """Drop the captured step (a graph that holds NCCL calls must be released
        before the process group is destroyed)."""
        self._graph = None

    def train(self) -> None:
        self._refuse_serving()
        for layer in self.layers:
            if hasattr(layer, "training"):
                layer.train()
        self._graph = None

    def eval(self) -> None:
        for layer in self.layers:
            if hasattr(layer, "training"):
                layer.eval()
        self._graph = None

    def __repr__(self):
        lines = ["Sequential("] + [f"  ({i}): {layer}" for i, layer in enumerate(self.layers)]
        return "\n".join(lines + [")"])

    def num_parameters(self) -> int:
        return sum(layer.num_parameters for layer in self.layers
                   if isinstance(layer, (LearnableLayer, Int8Linear)))

    def get_attention_scores(self) -> dict[int, tuple[Tensor, Tensor]]:
        out = {i: layer.get_attention_scores() for i, layer in enumerate(self.layers)
               if isinstance(layer, MultiheadAttentionV2)}
        if not out:
            raise RuntimeError("No attention layers in this Sequential.")
        return out
