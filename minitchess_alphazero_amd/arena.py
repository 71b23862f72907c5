"""Arena / gating: drop-in for the commented arena of exp/learner.py:97-145.

The reference's learner once played the new network against the previous one: its agent
first (RoundRobinReferee((new, old)): new moves first) then second, counted decisive games with
WinnerRecorder (exp/callbacks.py:7-28), and returned new_wins / (new_wins + old_wins + 1e-8);
LearnPuppet.update kept the new weights when that exceeded 0.55 (app/base.py:194-196, also
commented).  Here both sides run as batched engine play: the engine holds the two networks in
its two weight slots and each move's leaves are evaluated with the network of the agent to move
(mtaz_set_agent_slots).  All games of a side run in lockstep, so one launch per simulation wave
still covers every game.
"""
import numpy as np

ARENA_GAME_NUMBER_PER_SIDE = 3      # exp/learner.py:18
GATE = 0.55                         # app/base.py:195
DECISIVE = 1                        # csrc/rules.h Outcome


def winners(records):
    """WinnerRecorder.results over the games of one play(): {False: agent 0 wins, True: agent 1
    wins}; a decisive game is won by the agent that made the last move (exp/callbacks.py:19-22:
    winner = not referee.turn), draws are not counted."""
    res = {False: 0, True: 0}
    for plies, outcome in zip(records['plies'], records['outcome']):
        if int(outcome) == DECISIVE:
            res[bool((int(plies) - 1) % 2)] += 1
    return res


def arena(engine, new_net, old_net, seed_base=0):
    """Play engine.G games with the new network moving first and engine.G with it moving second.
    Returns {'new_wins', 'old_wins', 'draws', 'score'} with score as exp/learner.py:145.
    Afterwards weight slot 0 holds new_net and self-play (both agents on slot 0) is restored."""
    engine.set_weights(new_net, slot=0)
    engine.set_weights(old_net, slot=1)
    out = {'new_wins': 0, 'old_wins': 0, 'draws': 0, 'games': 0}
    try:
        for side, (s0, s1) in enumerate(((0, 1), (1, 0))):        # new first, then new second
            engine.set_agent_networks(s0, s1)
            engine.set_seed_base(seed_base + side * engine.G)
            engine.play()
            rec = engine.records()
            w = winners(rec)
            new_first = side == 0
            out['new_wins'] += w[False] if new_first else w[True]
            out['old_wins'] += w[True] if new_first else w[False]
            out['draws'] += int(np.sum(rec['outcome'] != DECISIVE))
            out['games'] += len(rec['plies'])
    finally:
        engine.set_agent_networks(0, 0)
    out['score'] = out['new_wins'] / (out['new_wins'] + out['old_wins'] + 1e-8)
    return out


def policy_match(new_net, old_net, games, device=0, seed=0, tau_change=6, repetition=1.0, frequency=0.0, presence=0.0):
    """New against old without search: every move is the mover's policy over its legal moves, sampled before
    fullmove tau_change and the likeliest one after (the schedule of exp/agent.py:114-118), in `games` games
    per side at once.  The penalties (logits.adjust_logits) weigh down actions the player has already
    taken in the game; 1, 0, 0 leave the policy as it is.  Returns arena()'s counts and score."""
    import torch

    from .engine import Engine
    from .environment import STARTING_FEN
    from .logits import adjust_logits, legal_masks
    if games < 1:
        raise ValueError(f'games must be at least 1, got {games}')
    dev = torch.device('cuda', device)
    rng = torch.Generator(device=dev).manual_seed(seed)
    engines = [Engine(n_games=games, sims=1, device=device) for _ in range(2)]   # the new and the old network
    out = {'new_wins': 0, 'old_wins': 0, 'draws': 0, 'games': 0}
    try:
        for eng, net in zip(engines, (new_net, old_net)):
            eng.set_weights(net)
        board = engines[0]                                        # which also holds the games
        for side in range(2):                                     # new first, then new second
            board.set_games([STARTING_FEN] * games)
            taken = [torch.empty((games, 0), dtype=torch.int32, device=dev) for _ in range(2)]   # by player
            pos, _, active, _ = board.games()
            ply = 0
            while active.any():
                player = ply % 2
                live = active.astype(bool)
                logits, _ = engines[player ^ side].evaluate_tensors(pos)
                adjust_logits(logits, legal=legal_masks(pos, dev), actions=taken[player], repetition=repetition,
                              frequency=frequency, presence=presence, out=logits)
                logits[torch.from_numpy(~live).to(dev)] = 0.0     # a finished game may have nothing legal
                if int(pos[live][0][4]) >> 16 < tau_change:       # the games move in lockstep
                    action = torch.multinomial(torch.softmax(logits, 1), 1, generator=rng)
                else:
                    action = logits.argmax(1, keepdim=True)
                taken[player] = torch.cat([taken[player], action.to(torch.int32)], 1)
                board.apply(action[:, 0].cpu().numpy())
                pos, _, active, outcome = board.games()
                ended = live & ~active.astype(bool)
                won = int(np.sum(outcome[ended] == DECISIVE))
                out['new_wins' if player == side else 'old_wins'] += won   # the last mover's (exp/callbacks.py:19-22)
                out['draws'] += int(ended.sum()) - won
                out['games'] += int(ended.sum())
                ply += 1
    finally:
        for eng in engines:
            eng.close()
    out['score'] = out['new_wins'] / (out['new_wins'] + out['old_wins'] + 1e-8)
    return out


def gate(score, threshold=GATE):
    """Keep the new network when it scored above the threshold (app/base.py:195-196)."""
    return score > threshold
