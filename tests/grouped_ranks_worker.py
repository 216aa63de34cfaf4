"""Worker of tests/test_gpu_grouped_ranks.py (not collected by pytest): ONE rank of a sharded run whose Adam phase is GroupedAdamW, on cuda:0.

    RANK=r WORLD_SIZE=n MASTER_ADDR=127.0.0.1 MASTER_PORT=p python grouped_ranks_worker.py <backend> <state_bits> <out.json>
"""
import json
import os
import sys

import numpy as np
import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

STEPS, MAX_NORM = 40, 1e-2


def main():
    backend, bits, out_path = sys.argv[1], int(sys.argv[2]), sys.argv[3]
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    dist.init_process_group(backend, rank=rank, world_size=world, **(dict(device_id=dev) if backend == "nccl" else {}))
    from pde_amd import scripts
    from pde_amd.optim import GroupedAdamW, grad_norm
    lb, ub = np.array([-10.0, -2.0]), np.array([10.0, 2.0])
    rng = np.random.default_rng(5)                # every rank draws the same data, the class shards the collocation points
    x0 = rng.uniform(lb[0], ub[0], (50, 1))
    data = x0, 1.0 / np.cosh(x0) ** 2, rng.uniform(lb[1], ub[1], (50, 1)), lb + (ub - lb) * rng.random((3001, 2))

    def trained(group, graph):
        torch.manual_seed(1234)
        m = scripts.kdv5_1soliton.PI.PhysicsInformedNN([2, 50, 50, 50, 50, 1], lb, ub, process_group=group)
        m.set_training_data(*data)
        m.adam_impl, m.adam_state_bits, m.max_grad_norm, m.use_hip_graph = "grouped", bits, MAX_NORM, graph
        m.train(STEPS, LBFGS_max_iter=0)
        return m

    res = {"rank": rank, "runs": {}}
    for name, group, graph in [("eager", dist.group.WORLD, False)] + ([("graph", dist.group.WORLD, True)] if backend == "nccl" else []) + [("single", None, False)]:
        m = trained(group, graph)
        if group is not None:
            m.check_replicas()
        opt = m.optimizer_Adam
        assert isinstance(opt, GroupedAdamW)
        theta = m.dnn.flat_theta().detach().cpu()
        run = {"steps": opt.device_state[:, 0].tolist(), "norm": float(opt.grad_norm), "theta": theta.numpy().tobytes().hex(),
               "state": [t.cpu().contiguous().view(torch.uint8).numpy().tobytes().hex() for t in (opt.exp_avg, opt.exp_avg_sq, opt.device_state)],
               "replays": getattr(m, "graph_stats", {}).get("replays", 0)}
        # one more closure and step: what the step reports is the norm of the whole closure's gradient, the same on every rank
        opt.zero_grad()
        m.backward()
        run["full_norm"] = float(grad_norm([p.grad for p in m.dnn.parameters()]))
        opt.step()
        run["step_norm"] = float(opt.grad_norm)
        res["runs"][name] = run
    with open(out_path, "w") as fh:
        json.dump(res, fh)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
