"""LoRA / DoRA adapter training: data loading, batching, masked next-token
loss, an Adam training loop with periodic validation and checkpointing.

Parity: LoRATrain (MLXLLM/LoraTrain.swift:134-433: Parameters :141, loss,
LoRABatchIterator, evaluate, train with progress callbacks, save) and
loadLoRAData (MLXLLM/Lora+Data.swift:21: ``.jsonl`` lines with a "text" field
or ``.txt`` lines). Resuming continues from ``completed_iterations`` with the
adapter weights the container already holds.

Loss: cross entropy of position j's logits against token j+1, counted only
where token j+1 is a real token of the sample (padding never scores).

With ``TrainParameters.fused`` the step runs on the training operators: the norms
around the blocks, counter-based dropout (a step's masks follow from the seed and the
step's number, resumed runs included) and the loss from the hidden rows without logits.
On CUDA the head's product takes its rows in bf16 there.
"""
from __future__ import annotations

import json
import os
import random
import time
from dataclasses import dataclass
from typing import Callable, Iterator

import torch
import torch.nn.functional as Fn

from .. import ops
from ..adapters.lora import LoRAContainer
from .forward import MaskStream, TrainableLoRA, train_forward, train_hidden


@dataclass
class TrainParameters:
    batch_size: int = 4
    iterations: int = 1000
    steps_per_report: int = 10
    steps_per_eval: int = 100
    validation_batches: int = 10  # 0 = the whole validation set
    save_every: int = 100
    adapter_path: str | None = None
    completed_iterations: int = 0
    learning_rate: float = 1e-5
    seed: int = 0
    fused: bool = False  # run on ops.block_norms, ops.dropout and ops.linear_cross_entropy

    def __post_init__(self):
        if self.completed_iterations < 0:
            raise ValueError("completed_iterations must be >= 0")


@dataclass
class Progress:
    kind: str  # "train" | "validation" | "save"
    iteration: int
    loss: float | None = None
    iterations_per_second: float | None = None
    tokens_per_second: float | None = None
    path: str | None = None


def load_lora_data(directory: str, name: str) -> list[str]:
    """``<directory>/<name>.jsonl`` (lines of {"text": ...}) or ``<name>.txt``."""
    for ext in ("jsonl", "txt"):
        p = os.path.join(directory, f"{name}.{ext}")
        if os.path.exists(p):
            return load_lora_file(p)
    raise FileNotFoundError(f"no {name}.jsonl or {name}.txt under {directory}")


def load_lora_file(path: str) -> list[str]:
    with open(path, encoding="utf-8") as f:
        lines = f.read().split("\n")
    if path.endswith(".jsonl"):
        out = []
        for ln in lines:
            if ln.startswith("{"):
                t = json.loads(ln).get("text")
                if t is not None:
                    out.append(t)
        return out
    return [ln for ln in lines if ln]


def iterate_batches(dataset: list[str], tokenizer, batch_size: int, train: bool,
                    seed: int = 0) -> Iterator[tuple[torch.Tensor, torch.Tensor, torch.Tensor]]:
    """(inputs [B, S-1], targets [B, S-1], lengths [B]) batches; endless and
    reshuffled each epoch when `train`, one pass otherwise."""
    rng = random.Random(seed)
    idx = list(range(len(dataset)))
    if train:
        rng.shuffle(idx)
    i = 0
    while True:
        if i >= len(idx):
            if not train:
                return
            rng.shuffle(idx)
            i = 0
        chunk = idx[i:i + batch_size]
        i += batch_size
        toks = [tokenizer.encode(dataset[j]) for j in chunk]
        lengths = [len(t) for t in toks]
        S = max(lengths)
        if S < 2:
            raise ValueError("LoRA batch has no sample of 2 or more tokens: each token is predicted from the "
                             "ones before it")
        arr = torch.zeros(len(toks), S, dtype=torch.long)
        for r, t in enumerate(toks):
            arr[r, :len(t)] = torch.tensor(t, dtype=torch.long)
        yield arr[:, :-1], arr[:, 1:], torch.tensor(lengths)


def loss_fn(model, lora: TrainableLoRA | None, inputs, targets, lengths, training=True, fused=False):
    """(mean loss over scored tokens, number of scored tokens). `fused`: from the
    hidden rows and the head, without logits."""
    S = inputs.shape[1]
    mask = torch.arange(S)[None, :] < (lengths[:, None] - 1)
    if fused:
        h = train_hidden(model, inputs, lora, training)
        if not isinstance(model.lm_head, torch.Tensor):
            raise ValueError("the fused loss needs a dense head")
        scored = torch.where(mask.to(h.device), targets.to(h.device), -100)
        loss = ops.linear_cross_entropy(h.to(model.lm_head.dtype), model.lm_head, scored,
                                        softcap=model.cfg.final_logit_softcap, reduction="mean")
        return loss, int(mask.sum())
    logits = train_forward(model, inputs, lora, training)
    mask = mask.to(logits.device)
    ce = Fn.cross_entropy(logits.reshape(-1, logits.shape[-1]), targets.to(logits.device).reshape(-1),
                          reduction="none").reshape(mask.shape)
    n = mask.sum()
    return (ce * mask).sum() / n.clamp_min(1), int(n)


@torch.no_grad()
def evaluate(model, lora, dataset, tokenizer, batch_size, batches=0, fused=False):
    tot, ntok = 0.0, 0
    for k, (x, y, ln) in enumerate(iterate_batches(dataset, tokenizer, batch_size, train=False)):
        if batches and k >= batches:
            break
        l, n = loss_fn(model, lora, x, y, ln, training=False, fused=fused)
        tot += float(l) * n
        ntok += n
    return tot / max(ntok, 1)


def train(model, adapter: LoRAContainer, tokenizer, train_set: list[str], valid_set: list[str],
          params: TrainParameters, progress: Callable[[Progress], bool] | None = None,
          optimizer_factory=None) -> LoRAContainer:
    """Train `adapter` on `train_set`; returns it with the trained weights.
    `progress` receives Progress events and may return False to stop."""
    lora = TrainableLoRA(adapter, model.embed.device)
    opt = (optimizer_factory or (lambda ps: torch.optim.Adam(ps, lr=params.learning_rate)))(list(lora.parameters()))
    it = iterate_batches(train_set, tokenizer, params.batch_size, train=True, seed=params.seed)
    losses, ntoks = [], 0
    t0 = time.perf_counter()
    start = params.completed_iterations
    for step in range(start, params.iterations):
        x, y, ln = next(it)
        if params.fused:
            lora.masks = MaskStream(params.seed, step)
        loss, n = loss_fn(model, lora, x, y, ln, training=True, fused=params.fused)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
        ntoks += n
        i = step + 1
        if i % params.steps_per_report == 0:
            dt = time.perf_counter() - t0
            ev = Progress("train", i, sum(losses) / len(losses), params.steps_per_report / dt, ntoks / dt)
            losses, ntoks = [], 0
            t0 = time.perf_counter()
            if progress and progress(ev) is False:
                break
        if valid_set and (i == 1 or i % params.steps_per_eval == 0):
            vl = evaluate(model, lora, valid_set, tokenizer, params.batch_size, params.validation_batches, params.fused)
            if progress and progress(Progress("validation", i, vl)) is False:
                break
        if params.adapter_path and i % params.save_every == 0:
            lora.write_back()
            adapter.save(params.adapter_path)
            if progress and progress(Progress("save", i, path=params.adapter_path)) is False:
                break
    lora.write_back()
    if params.adapter_path:
        adapter.save(params.adapter_path)
    return adapter
