"""The way of the prefill kernel's row threads through their items (csrc/kv8_walk.cuh), gone on the CPU with waits that run out at every
place: nobody is left waiting at a meeting.  A thread here is a warp there: two groups of two for each row of the tile."""
import shutil
import subprocess
from pathlib import Path

import pytest

from esp_b200.csrc.build import CSRC

HARNESS = r"""
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <thread>
#include <vector>
#include WALK

// a named barrier with a conjunction: nobody leaves before ``count`` have come
struct Meeting {
    int count, here = 0, turn = 0;
    bool all = true, said = true;
    std::mutex m;
    std::condition_variable c;
    bool operator()(bool ok) {
        std::unique_lock<std::mutex> lock(m);
        all = all && ok;
        const int mine = turn;
        if (++here == count) {
            said = all, here = 0, all = true, turn++;
            c.notify_all();
            return said;
        }
        if (!c.wait_for(lock, std::chrono::seconds(30), [&] { return turn != mine; })) {
            std::printf("a meeting of %d waits for %d\n", count, count - here);
            std::fflush(stdout);
            std::_Exit(1);
        }
        return said;
    }
};

// an item: 0 two tiles, two blocks each; n > 0: one tile of n blocks, which the groups take in turn
static bool run(const std::vector<int>& items, const int (&fails)[2][2]) {
    Meeting group[2] = {{2}, {2}}, across{4};
    std::vector<int> finished[2][2];
    bool whole[2][2];
    auto warp = [&](int g, int side) {
        int now = -1, waits = 0;
        auto wait = [&] { return waits++ < fails[g][side]; };          // the first that runs out and all behind it
        auto open = [&](int round) {
            now = round;
            return round < (int)items.size();
        };
        auto two_tiles = [&] { return items[now] == 0; };
        auto work = [&] {
            const int blocks = items[now] == 0 ? 2 : (items[now] + 1 - g) / 2;
            for (int j = 0; j < blocks; j++)
                if (!group[g](wait())) return false;
            return wait();
        };
        auto meet = [&](bool all_groups, bool ok) { return all_groups ? across(ok) : group[g](ok); };
        auto finish = [&] { finished[g][side].push_back(now); };
        whole[g][side] = kv8_walk_items(open, two_tiles, work, meet, finish);
    };
    std::vector<std::thread> threads;
    for (int g = 0; g < 2; g++)
        for (int side = 0; side < 2; side++) threads.emplace_back(warp, g, side);
    for (auto& t : threads) t.join();
    // an item of one tile is finished by all or by none; whoever goes the whole way has finished all
    for (int i = 0; i < (int)items.size(); i++) {
        int n = 0;
        for (auto& f : finished)
            for (auto& list : f)
                for (int done : list) n += done == i;
        if (items[i] > 0 && n != 0 && n != 4) return false;
    }
    for (int g = 0; g < 2; g++)
        for (int side = 0; side < 2; side++)
            if (whole[g][side] != (finished[g][side].size() == items.size())) return false;
    return true;
}

int main() {
    const int kinds[] = {0, 1, 2, 3}, never = 1 << 20;
    long runs = 0;
    for (int length = 1; length <= 3; length++) {
        int patterns = 1;
        for (int i = 0; i < length; i++) patterns *= 4;
        for (int pattern = 0; pattern < patterns; pattern++) {
            std::vector<int> items;
            for (int i = 0, x = pattern; i < length; i++, x /= 4) items.push_back(kinds[x % 4]);
            for (int a = 0; a <= 3 * length; a++)
                for (int b = 0; b <= 3 * length; b++)
                    for (int one_side = 0; one_side < 2; one_side++) {
                        const int fa = a == 3 * length ? never : a, fb = b == 3 * length ? never : b;
                        const int fails[2][2] = {{fa, one_side ? never : fa}, {one_side ? never : fb, fb}};
                        if (!run(items, fails)) {
                            std::printf("items finished by some alone\n");
                            return 1;
                        }
                        runs++;
                    }
        }
    }
    std::printf("%ld\n", runs);
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_nobody_is_left_at_a_meeting(tmp_path: Path):
    (tmp_path / "walk.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", f'-DWALK="{CSRC / "kv8_walk.cuh"}"', str(tmp_path / "walk.cpp"), "-o", str(tmp_path / "walk")],
                   check=True)
    got = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stdout
    assert int(got.stdout) == 2 * (4 * 4 ** 2 + 16 * 7 ** 2 + 64 * 10 ** 2)
