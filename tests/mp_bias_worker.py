"""Child process of tests/test_sync_bias.py: one gloo rank of several that step
the balance bias of their experts together.

On the CPU the communicator, the Collective operator and the bias' kernel have
stand-ins (the operator's adds up over gloo); on GPUs, one for each rank,
everything is the framework's."""

import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

NUM, RATE = 5, 0.25
CALLS = []


def counts_of(rank):
    return [3 * rank + 1, 7, 2 * (rank % 2), 11 - 3 * rank, 4]


def stand_ins(rank):
    import torch
    import torch.distributed as dist
    import dragon_b200.comm as comm_module
    from dragon_b200 import experts, gradient_sync
    from dragon_b200.distributed import backend
    from tests.mp_worker import FakeCommunicator
    comm_module.Communicator = FakeCommunicator
    backend._TorchWorld.device = lambda self: 0

    def execute(group, inputs, outputs=None, **args):
        CALLS.append("all-reduce")
        assert args == {"operation": "ALLREDUCE", "reduction": "SUM"}
        assert len(inputs) == 1 and outputs is not None and outputs[0] is inputs[0] and inputs[0].dtype == torch.int32
        if group.size > 1:
            dist.all_reduce(inputs[0])

    def update_bias(bias, counts, rate, out=None):
        CALLS.append("update")
        lack = counts.sum().item() - NUM * counts.long()
        return bias.add_(rate * lack.sign().float())

    gradient_sync._execute, experts.update_bias = execute, update_bias


def main():
    where, rank, world, port = sys.argv[1], int(sys.argv[2]), int(sys.argv[3]), sys.argv[4]
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=port, RANK=str(rank), WORLD_SIZE=str(world))
    import torch
    import torch.distributed as dist
    dist.init_process_group(backend="gloo", rank=rank, world_size=world)
    if where == "gpu":
        torch.cuda.set_device(rank)
        device = torch.device("cuda", rank)
    else:
        stand_ins(rank)
        device = torch.device("cpu")
    from dragon_b200.distributed import backend
    from dragon_b200.gradient_sync import sync_expert_bias
    everyone = backend.new_group(list(range(world)))
    last = backend.new_group([world - 1])
    start = torch.arange(NUM, dtype=torch.float32) / 8
    total = [sum(c) for c in zip(*(counts_of(r) for r in range(world)))]

    def step(counts):
        return [b + RATE * ((c * NUM < sum(counts)) - (c * NUM > sum(counts))) for b, c in zip(start.tolist(), counts)]

    def call(group, default=None):
        del CALLS[:]
        bias, counts = start.clone().to(device), torch.tensor(counts_of(rank), dtype=torch.int32, device=device)
        if default is None:
            assert sync_expert_bias(bias, counts, RATE, group) is bias
        else:
            with default.as_default():
                assert sync_expert_bias(bias, counts, RATE) is bias
        return bias.tolist(), counts.tolist()

    # The group's counts, by an all-reduce before the update, and the same bias on every rank.
    for result in (call(everyone), call(None, everyone)):
        assert result == (step(total), total), result
        assert where == "gpu" or CALLS == ["all-reduce", "update"]
    # A group of one rank: its own counts there, nothing at all on the others.
    bias, counts = call(last)
    assert counts == counts_of(rank)
    assert bias == (step(counts) if rank == world - 1 else start.tolist())
    assert where == "gpu" or bool(CALLS) == (rank == world - 1)
    # Without a group each rank counts for itself.
    assert call(None) == (step(counts_of(rank)), counts_of(rank))
    assert where == "gpu" or CALLS == ["update"]
    dist.barrier()
    backend.finalize()
    dist.destroy_process_group()
    print("WORKER_OK", rank)


if __name__ == "__main__":
    main()
