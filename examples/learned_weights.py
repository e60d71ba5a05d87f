"""Learns to read a vehicle's tracking weights from its history.

Each of a batch of point masses is driven by an expert with control and final-state weights
of its own, which nobody tells us: all there is, is a recorded trajectory.  A history
model (turbompc_amd.learning) maps the record to weights, the differentiable solve
turns the weights into controls from another start, and the error against the expert's
controls there flows back through the solve into the model.  Afterwards the model runs as
a control loop would run it, one record row per period.

    python3 examples/learned_weights.py
"""
from __future__ import annotations

import copy
import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from turbompc_amd.learning import HistoryWeights
from turbompc_amd.problems import configs
from turbompc_amd.solvers.turbompc_solver import DEFAULT_SOLVER_PARAMS, TurboMPCSolver

CONTROL, FINAL = "weights_penalization_control_squared", "weights_penalization_final_state"


def run(B: int = 256, steps: int = 60, width: int = 64, dtype: torch.dtype = torch.float32, seed: int = 0, say=print,
        **options):
    """(losses, the model, histories, lengths) of a short training run; options: the model's memory, norm and dropout."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    torch.manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=gen, device=dev, dtype=torch.float64)  # noqa: E731
    prob = configs.config1(B=B, seed=seed).to(dev, torch.float64)
    params = copy.deepcopy(DEFAULT_SOLVER_PARAMS)
    params["num_sqp_iteration_max"] = 1
    params["admm"].update(max_iter=50, adapt_rho_every=0)
    solver = TurboMPCSolver(prob, params)
    guess = solver.initial_guess()

    # the experts, their records (ragged: at least 5 steps) and what they do from a new start
    expert = {CONTROL: 10.0 ** (2 * rand(B, 1) - 1.5).expand(B, 2), FINAL: 1.0 + 9.0 * rand(B, 4)}
    record = solver.solve(guess, {"initial_state": 2 * rand(B, 4) - 1}, expert)
    history = torch.cat([record.states, record.controls], dim=-1)
    lengths = torch.randint(5, history.shape[1] + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
    start = {"initial_state": 2 * rand(B, 4) - 1}
    target = solver.solve(guess, start, expert).controls[:, :-1]

    model = HistoryWeights(history.shape[-1], {CONTROL: 2, FINAL: 4}, width=width, layers=2, heads=4, kv_heads=2,
                           hidden=3 * width, dtype=dtype, device=dev, **options)
    key = torch.tensor([seed, 0], device=dev)  # of the masks, where the model drops
    solve = solver.get_differentiable_solve_function()
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for i in range(steps):
        weights = {k: w.double() for k, w in model(history, lengths, key).items()}
        controls = solve(guess, start, weights).controls[:, :-1]
        loss = ((controls - target) ** 2).mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        key[1] += 1
        losses.append(loss.detach())
        if i % 10 == 0 or i + 1 == steps:
            say(f"step {i:4d}  mean squared control error {float(loss.detach()):.5f}")
    return torch.stack(losses).tolist(), model.eval(), history, lengths


def control_loop(model, history, lengths):
    """The weights of every problem after its last record row, row by row."""
    state = model.initial_state(history.shape[0])
    last = None
    for t in range(history.shape[1]):
        active = lengths > t
        w = model.step(history[:, t], state, active)
        last = w if last is None else {k: torch.where(active[:, None], w[k], last[k]) for k in w}
    return last


if __name__ == "__main__":
    _, model, history, lengths = run()
    with torch.no_grad():
        whole = model(history, lengths)
    looped = control_loop(model, history, lengths)
    worst = max(float((whole[k] - looped[k]).abs().max() / whole[k].abs().max()) for k in whole)
    print(f"row by row against the whole history: {worst:.1e} of the largest weight apart")
