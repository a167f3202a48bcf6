"""Energies of a batch of structures from ACE features, species vectors and attention among the atoms.

    python examples/attention_energies.py [--steps 30]

The ACE features of every atom (fixed, from ``ACEEvaluator``) and a learned vector of its species
(``runtime.species_embedding``) make its state; one attention layer exchanges states among the atoms of each
structure, weaker with distance (``runtime.structure_attention``); a second one, with a single query per structure,
pools them into an energy.  The model is fitted to energies of a pair potential, which the features alone, with
their cutoff, describe in part.  The features' neighbours are those of a periodic box; the attention and the energies
know the atoms in it and none of their images.
"""

import argparse
import os
import sys

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if REPO not in sys.path:
    sys.path.insert(0, REPO)

from ye3t_b200 import runtime  # noqa: E402
from ye3t_b200.ace import ACEConfig, ACEEvaluator  # noqa: E402
from ye3t_b200.schedules import ACEBundle  # noqa: E402

HEADS, WIDTH, SPECIES = 4, 32, 3
CHANNELS = HEADS * WIDTH


class AttentionEnergies(torch.nn.Module):
    def __init__(self, features, device):
        super().__init__()
        make = {"device": device, "dtype": torch.float32}
        self.table = torch.nn.Parameter(torch.randn(SPECIES, CHANNELS, **make))
        self.project = torch.nn.Linear(features, CHANNELS, **make)
        self.qkv = torch.nn.Linear(CHANNELS, 3 * CHANNELS, bias=False, **make)
        self.pool_query = torch.nn.Parameter(torch.zeros(1, HEADS, WIDTH, **make))  # starts as the mean
        self.pool = torch.nn.Linear(CHANNELS, 2 * CHANNELS, bias=False, **make)
        self.energy = torch.nn.Linear(CHANNELS, 1, **make)
        # heads from local to long-ranged: decay per Angstrom
        self.slopes = torch.nn.Parameter(2.0 ** -torch.arange(HEADS, **make))

    def forward(self, features, species, positions, atoms, pooled):
        """Energy per atom of every structure; ``atoms`` and ``pooled`` are the batch's layouts."""
        state = self.project(features) + runtime.species_embedding(self.table, species, scale=CHANNELS ** -0.5)
        q, k, v = self.qkv(state).view(-1, 3, HEADS, WIDTH).unbind(1)
        state = state + runtime.structure_attention(q, k, v, atoms, positions=positions,
                                                    slopes=self.slopes).reshape(state.shape)
        k, v = self.pool(state).view(-1, 2, HEADS, WIDTH).unbind(1)
        query = self.pool_query.expand(pooled.query_count, HEADS, WIDTH)
        return self.energy(runtime.structure_attention(query, k, v, pooled).reshape(-1, CHANNELS))[:, 0]


def structures(counts, device, seed=0):
    """Random boxes at 0.05 atoms per cubic Angstrom: positions, species, ACE features and standardised pair
    energies per atom."""
    bundle = ACEBundle.load(os.path.join(REPO, "ye3t_b200", "bundles", "ace_n8_l3_nu3_L0.npz"))
    ev = ACEEvaluator(bundle, device, config=ACEConfig(5.0, 5.0), species_prefactor=[1.0, 0.75, 1.25])
    g = torch.Generator(device=device).manual_seed(seed)
    batch = []
    for n in counts:
        box = (n / 0.05) ** (1.0 / 3.0)
        x = torch.rand(n, 3, generator=g, device=device, dtype=torch.float64) * box
        z = torch.randint(0, SPECIES, (n,), generator=g, device=device, dtype=torch.int32)
        rows, neighbors = ev.neighbor_list(x, box)
        b = ev.features(ev.density(x, z, box, rows, neighbors)).real
        apart = (x[:, None] - x[None]).norm(dim=-1) + torch.eye(n, device=device) * 1e9
        charge = z.double() - 1.0
        energy = (charge[:, None] * charge[None] * torch.exp(-apart / 4.0)).sum() / n
        batch.append((x, z, b, energy))
    x, z, b, e = (torch.cat([s[k].reshape(-1, *s[k].shape[1:]) if k < 3 else s[k][None] for s in batch])
                  for k in range(4))
    b = (b - b.mean(0)) / b.std(0).clamp_min(1e-12)
    return x.float(), z, b.float(), ((e - e.mean()) / e.std()).float()


def train(steps, device="cuda:0", counts=(300, 80, 150, 33, 512, 64), log=print):
    torch.manual_seed(0)
    x, z, features, target = structures(counts, device)
    model = AttentionEnergies(features.shape[1], device)
    atoms = runtime.StructureLayout(counts, heads=HEADS, device=device)
    pooled = runtime.StructureLayout([1] * len(counts), counts, heads=HEADS, device=device)
    adam = torch.optim.Adam(model.parameters(), lr=3e-4)
    losses = []
    for step in range(steps):
        loss = (model(features, z, x, atoms, pooled) - target).square().mean()
        adam.zero_grad()
        loss.backward()
        adam.step()
        losses.append(loss.detach())
        if log and step % 10 == 0:
            log(f"step {step:3d}  mean squared error {float(losses[-1]):.6f}")
    x.requires_grad_(True)
    energy = (model(features, z, x, atoms, pooled) * torch.tensor(counts, device=device)).sum()
    (forces,) = torch.autograd.grad(-energy, x)
    return [float(v) for v in losses], forces


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=30)
    losses, forces = train(parser.parse_args().steps)
    print(f"mean squared error {losses[0]:.6f} -> {losses[-1]:.6f}; attention's share of the forces: "
          f"{float(forces.norm(dim=1).mean()):.6f} per atom")


if __name__ == "__main__":
    main()
